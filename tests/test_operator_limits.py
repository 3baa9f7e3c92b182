"""Limits of the linear entry points that need no GPU: the width from which sums in the tensor cores that are
not drained on the way would lose more than an fp16 output's rounding."""
import ctypes

from brimkern_b200 import _lib as L


def test_inner_widths_of_undrained_sums():
    stand_in = ctypes.create_string_buffer(4096)
    a = (ctypes.addressof(stand_in) + 15) // 16 * 16
    lib = L.lib()
    # No rows: accepted widths do nothing, before any tensor is looked at.
    linear = lambda k, t: lib.brk_linear(a, 0, k, 8, None, None, None, 0, None, None, t, None)  # noqa: E731
    gate_up = lambda k: lib.brk_ffn_gate_up(a, 0, k, 8, None, None, None, None, None, 1, None, None)  # noqa: E731
    ffn = lambda d, ff: lib.brk_ffn(a, 0, d, ff, None, None, 1e-6, 0, None, None, None, None, 1, None, None)  # noqa: E731
    w, m = 1 << 24, 1 << 15
    assert linear(w, L.BRK_T_F16) == linear(w, L.BRK_T_F32) == gate_up(m) == ffn(m, w) == L.BRK_OK
    for rc in (linear(w + 8, L.BRK_T_F16), linear(w + 8, L.BRK_T_F32), gate_up(m + 8), ffn(m + 8, 64), ffn(64, w + 8),
               linear(64, 2)):
        assert rc == L.BRK_ERR_INVALID
