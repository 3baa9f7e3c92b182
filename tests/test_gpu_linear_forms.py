"""The linear operators on shapes that reach every form that a product is cut into -- one CTA or a CTA pair
to a tile; tiles whole, their k split over a cluster, or dealt as ranges of (tile, k step) units, first or
after whole waves; f32 outputs with more than one accumulator set to a piece -- against 64 bits.
tests/test_linear_plan.py checks, without a GPU, that these shapes are cut like that.  Tolerances:
tests/test_gpu_linear.py."""
import math

import pytest

from test_gpu_linear import act64, assert_within, inputs, product64, rounded

pytestmark = pytest.mark.gpu

# (CTAs to a tile, cut), rows, k, n.  f32 outputs of all of them drain.
LINEAR = [
    (("one", "whole"), 44, 1744, 7495),
    (("one", "whole"), 103, 1096, 5001),
    (("one", "cluster"), 80, 10240, 2560),
    (("one", "cluster"), 150, 10240, 2560),
    (("one", "ranged"), 52, 9440, 10051),
    (("pair", "whole"), 320, 1112, 7014),
    (("pair", "cluster"), 300, 4096, 2560),
    (("pair", "cluster"), 400, 10240, 2560),
    (("pair", "cluster"), 600, 2560, 2560),
    (("pair", "ranged"), 2000, 2560, 2560),
    (("pair", "ranged"), 2048, 10240, 2560),
    (("pair", "ranged"), 1823, 6280, 1217),
    (("pair", "ranged after whole"), 1156, 6280, 8505),
]
GATE_UP = [
    (("one", "cluster"), 77, 2304, 1215),
    (("one", "ranged"), 10, 8760, 75),
    (("one", "ranged"), 85, 4760, 9636),
    (("one", "ranged after whole"), 1395, 5760, 7975),
    (("pair", "cluster"), 291, 1048, 1003),
    (("pair", "whole"), 600, 2560, 2560),
    (("pair", "ranged"), 89, 3024, 9665),
    (("pair", "ranged after whole"), 243, 1784, 9530),
]


@pytest.mark.parametrize("form,rows,k,n", LINEAR)
def test_linear_f32(eng, form, rows, k, n):
    """Without and with bias, activation and residual (in place), and the same bits every time."""
    import torch
    rnd, x, w = inputs(eng, rows + k + n, rows, k, n)
    b, r = 0.1 * rnd(n), 2.0 * rnd(rows, n)
    y, err = product64(x, w, None, True)
    first = eng.linear(x, w, torch.full((rows, n), float("nan"), device=eng.device))
    assert_within(first, y, rounded(y, err, first.dtype), "plain")
    for _ in range(30):
        assert torch.equal(eng.linear(x, w, torch.empty_like(first)), first)
    z = act64(y + b.double(), "silu") + r.double()
    tol = 1.13 * (err + 2.0 ** -23 * (y + b.double()).abs()) + 2.0 ** -20 * y.abs() + 2.0 ** -22 * (z.abs() + r.double().abs())
    out = r.clone()
    assert_within(eng.linear(x, w, out, bias=b, act="silu", residual=out), z, rounded(z, tol, out.dtype), "residual")
    eng.ctx.check()


@pytest.mark.parametrize("form,rows,k,n", LINEAR)
def test_linear_fp16(eng, form, rows, k, n):
    import torch
    rnd, x, w = inputs(eng, rows + k + n, rows, k, n)
    r = 2.0 * rnd(rows, n)
    y, err = product64(x, w, None, False)
    first = eng.linear(x, w, torch.full((rows, n), float("nan"), dtype=torch.float16, device=eng.device))
    assert_within(first, y, rounded(y, err, first.dtype), "plain")
    z = y + r.double()
    out = eng.linear(x, w, torch.empty_like(first), residual=r)
    assert_within(out, z, rounded(z, err + 2.0 ** -23 * z.abs(), out.dtype), "residual")
    for _ in range(10):
        assert torch.equal(eng.linear(x, w, torch.empty_like(first)), first)
    eng.ctx.check()


@pytest.mark.parametrize("form,rows,k,n", GATE_UP)
def test_gate_up(eng, form, rows, k, n):
    import torch
    rnd, x, w = inputs(eng, rows * 3 + k + n, rows, k, n)
    u = (rnd(n, k) / math.sqrt(k)).half()
    bg, bu = 0.3 * rnd(n), 0.3 * rnd(n)
    gate, eg = product64(x, w, bg, False)
    up, eu = product64(x, u, bu, False)
    a = act64(gate, "silu")
    ref = a * up
    tol = (1.13 * eg + 2.0 ** -20 * gate.abs()) * up.abs() + a.abs() * eu + eg * eu * 2 + 2.0 ** -22 * ref.abs()
    first = eng.ffnGateUp(x, w, u, torch.full((rows, n), float("nan"), dtype=torch.float16, device=eng.device), b_gate=bg, b_up=bu)
    assert_within(first, ref, rounded(ref, tol, first.dtype), "gate-up")
    for _ in range(10):
        assert torch.equal(eng.ffnGateUp(x, w, u, torch.empty_like(first), b_gate=bg, b_up=bu), first)
    eng.ctx.check()


@pytest.mark.parametrize("rows", [80, 400])
def test_ffn_block(eng, rows):
    """The whole block at an FFN's widths: the way back drains its accumulators (tolerance:
    tests/test_gpu_linear.py's test_ffn_block)."""
    import torch
    d, ff = 2560, 10240
    rnd, _, wg = inputs(eng, 17, 1, d, ff)
    wu, wd = (rnd(ff, d) / math.sqrt(d)).half(), (rnd(d, ff) / math.sqrt(ff)).half()
    h, norm = 3.0 * rnd(rows, d), 1 + 0.1 * rnd(d)
    out = torch.full((rows, d), float("nan"), device=eng.device)
    eng.ffn(h, wg, wu, wd, out, ffn_norm=norm)
    eng.ctx.check()
    h64 = h.double()
    x = h64 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + 1e-6) * norm.double()
    y = (act64(x @ wg.double().t(), "silu") * (x @ wu.double().t())) @ wd.double().t()
    ref = h64 + y
    size = y.pow(2).mean(-1, keepdim=True).sqrt()
    tol = 6 * 2.2 * 2.0 ** -11 / math.sqrt(3) * size + 2.0 ** -22 * ref.abs() + 1e-5
    assert_within(out, ref, tol, "ffn")
    for _ in range(10):
        assert torch.equal(eng.ffn(h, wg, wu, wd, torch.empty_like(out), ffn_norm=norm), out)


@pytest.mark.parametrize("k", [16384, 16392, 65536])
def test_wide_fp16_sums_lose_nothing(eng, k):
    """Operands of one sign, whole tiles of k: the tensor cores' truncation is a bias of the sum, at most
    k / 16 steps of 2^-23 without a drain (5.9e-9 of the sum for each of k seen: 1e-4 at the last undrained
    width), 64 steps with one.  The mean over many outputs averages their own rounding out (2^-11 / sqrt(3 *
    65536) = 1.1e-6)."""
    import torch
    g = torch.Generator(device=eng.device).manual_seed(k)
    rows, n = 512, 9472
    x = torch.rand((rows, k), generator=g, device=eng.device, dtype=torch.float16) / 64
    w = torch.empty((n, k), dtype=torch.float16, device=eng.device)
    for part in w.split(1184):
        part.copy_(torch.rand(part.shape, generator=g, device=eng.device) * 256 / k)
    y = eng.linear(x, w, torch.empty((rows, n), dtype=torch.float16, device=eng.device))
    eng.ctx.check()
    ref = x[:128].double() @ w[-512:].double().t()
    lost = abs(((y[:128, -512:].double() - ref) / ref).mean().item())
    assert lost <= (1.2e-4 if k <= 16384 else 64 * 2.0 ** -23 + 4 * 1.1e-6), lost
