"""Refusals of the shared-prefix and linear entry points that need no GPU: null handles and bad
scalars come back as a status before anything is touched, and the Python layer names the tensor it
refuses."""
import ctypes

import pytest

from brimkern_b200 import _lib as L


def _past(*v):
    return (ctypes.c_int32 * len(v))(*v)


def test_null_handles_are_refused():
    lib = L.lib()
    p = L.AttnParams(8, 8, 64, 0.0, 0.0, 0, 0, 0, 1e-6, None, None, None)
    assert lib.brk_attn_decode_prefix(None, None, 0, 0, None, 0, ctypes.byref(p), 1, 1, _past(0), None, 0, None, 0,
                                      None) == L.BRK_ERR_INVALID
    assert lib.brk_attn_step_prefix(None, None, 0, 0, None, 0, ctypes.byref(p), 1, 1, _past(0), None, None, None, None,
                                    None, 0, None) == L.BRK_ERR_INVALID
    assert lib.brk_linear(None, 1, 64, 1, None, None, None, 0, None, None, 0, None) == L.BRK_ERR_INVALID
    assert lib.brk_ffn_gate_up(None, 1, 64, 1, None, None, None, None, None, 0, None, None) == L.BRK_ERR_INVALID
    assert lib.brk_ffn(None, 1, 64, 64, None, None, 1e-6, 0, None, None, None, None, 0, None, None) == L.BRK_ERR_INVALID


@pytest.mark.parametrize("rows,k,n,act,out_type", [
    (-1, 64, 8, 0, 0), (1, 0, 8, 0, 0), (1, 60, 8, 0, 0), (1, -8, 8, 0, 0), (1, 64, 0, 0, 0), (1, 64, -4, 0, 0),
    (1, 64, 8, 5, 0), (1, 64, 8, -1, 0), (1, 64, 8, 0, 2), (2 ** 31 - 1, 64, 2 ** 31 - 1, 0, 0), (2 ** 31 - 1, 8, 1, 0, 0),
    (1, 8, 2 ** 31 - 1, 0, 0), (1, 8, 2 ** 30 + 1, 0, 0)])
def test_linear_scalars_are_refused(rows, k, n, act, out_type):
    """The checks run before the context or a tensor is looked at: stand-ins do."""
    stand_in = ctypes.create_string_buffer(4096)
    a = (ctypes.addressof(stand_in) + 15) // 16 * 16
    rc = L.lib().brk_linear(a, rows, k, n, a, a + 512, None, act, None, a + 1024, out_type, None)
    assert rc in (L.BRK_ERR_INVALID, L.BRK_ERR_CAPACITY)
    if out_type == 0:
        rc = L.lib().brk_ffn_gate_up(a, rows, k, n, a, a + 512, a + 512, None, None, act, a + 1024, None)
        assert rc in (L.BRK_ERR_INVALID, L.BRK_ERR_CAPACITY)


def test_linear_pointers_are_refused():
    stand_in = ctypes.create_string_buffer(1 << 16)
    a = (ctypes.addressof(stand_in) + 15) // 16 * 16
    lib = L.lib()
    x, w, o = a, a + 1024, a + 8192
    for args in ((0, w, None, None, o), (x, 0, None, None, o), (x, w, None, None, 0), (x + 2, w, None, None, o),
                 (x, w + 2, None, None, o), (x, w, None, None, o + 2), (x, w, None, None, x), (x, w, None, None, w + 64),
                 (x, w, o, None, o), (x, w, None, o + 4, o), (x, w, a + 16386, None, o), (x, w, None, a + 16386, o)):
        assert lib.brk_linear(a, 2, 64, 8, args[0], args[1], args[2], 0, args[3], args[4], 0, None) == L.BRK_ERR_INVALID
    for b_gate, b_up in ((a + 16386, None), (None, a + 16385)):
        assert lib.brk_ffn_gate_up(a, 2, 64, 8, x, w, w, b_gate, b_up, 0, o, None) == L.BRK_ERR_INVALID


def test_zero_rows_do_nothing():
    stand_in = ctypes.create_string_buffer(64)
    assert L.lib().brk_linear(ctypes.addressof(stand_in), 0, 64, 8, None, None, None, 0, None, None, 0, None) == L.BRK_OK


def test_python_layer_names_the_tensor():
    torch = pytest.importorskip("torch")
    from brimkern_b200.engine import AttentionEngine
    eng = AttentionEngine.__new__(AttentionEngine)  # the checks need no context
    eng.device = torch.device("cpu")
    t = torch.zeros((4, 8), dtype=torch.float16)
    assert eng._tensor(t, "t", (torch.float16,), (4, 8)) == t.data_ptr()
    for bad, word in ((t.float(), "float32"), (t[:, ::2], "contiguous"), (t.view(8, 4), "shape")):
        with pytest.raises(L.BrkError, match=word):
            eng._tensor(bad, "t", (torch.float16,), (4, 8) if word == "shape" else None)
    eng.device = torch.device("cuda", 0)
    with pytest.raises(L.BrkError, match="on cpu"):
        eng._tensor(t, "t", (torch.float16,), None)
    with pytest.raises(L.BrkError, match="activation"):
        eng._activation("tanh")
