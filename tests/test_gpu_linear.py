"""The linear operators on fp16 activations (brk_linear, brk_ffn_gate_up, brk_ffn) against 64 bits.

Tolerance, from the arithmetic: a product sum takes K / 16 tensor-core steps, each truncated by at
most 2^-22 of A = sum |x w| (the running sum never exceeds it; the products' alignment costs as
much again, hence 2^-22 and not 2^-23).  brk_linear's accumulators hold 1024 of k at most and the
parts are added in f32, so its sums are off by at most (64 * 2^-22 + parts * 2^-24) A; gate-up's by
K / 16 * 2^-22 A.  The activations have a slope of at most 1.13 and cost a few 2^-24 of their own;
bias, product and residual one rounding each; an fp16 output half a step, 2^-11 of the value (or
2^-25 below the normal range)."""
import math

import pytest

pytestmark = pytest.mark.gpu

ACTS = ["none", "silu", "gelu", "gelu_tanh", "quick_gelu"]


def act64(x, act):
    import torch
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    if act == "quick_gelu":
        return x * torch.sigmoid(1.702 * x)
    return x


def product64(x, w, b, drained):
    """x w^T + b in 64 bits and the bound of the kernel's error in it."""
    y = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    k = x.shape[1]
    steps = min(k, 1024) / 16 if drained else k / 16
    err = mag * ((steps + 2) * 2.0 ** -22 + (k / 64 + 2) * 2.0 ** -24)
    if b is not None:
        y = y + b.double()
        err = err + 2.0 ** -23 * y.abs()
    return y, err


def rounded(y, err, dtype):
    import torch
    if dtype == torch.float16:
        return err * (1 + 2.0 ** -10) + 2.0 ** -11 * y.abs() + 2.0 ** -25
    return err + 2.0 ** -23 * y.abs() + 1e-37


def assert_within(got, ref, tol, what):
    import torch
    torch.cuda.synchronize()
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {(err / tol).max().item():.3g} of "
                           f"the tolerance at {tuple(int(i) for i in bad.nonzero()[0])}")


def inputs(eng, seed, rows, k, n):
    import torch
    g = torch.Generator(device=eng.device).manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=eng.device)  # noqa: E731
    return rnd, rnd(rows, k).half(), (rnd(n, k) / math.sqrt(k)).half()


SHAPES = [(1, 8, 1), (1, 64, 128), (1, 4096, 2560), (3, 72, 129), (16, 1000, 127), (17, 1024, 257), (31, 2048, 640),
          (33, 136, 5), (64, 2560, 1030), (65, 520, 383), (77, 2304, 515), (128, 1024, 128), (129, 1032, 1000),
          (255, 64, 300), (256, 256, 256), (257, 1024, 4096), (300, 4104, 130), (511, 200, 700), (1000, 2560, 384),
          (5, 10240, 2560), (130, 10240, 300)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear_shapes(eng, rows, k, n):
    import torch
    rnd, x, w = inputs(eng, rows + k + n, rows, k, n)
    b, r = 0.1 * rnd(n), 2.0 * rnd(rows, n)
    y, err = product64(x, w, None, True)
    out = torch.full((rows, n), float("nan"), device=eng.device)
    assert_within(eng.linear(x, w, out), y, rounded(y, err, out.dtype), "plain f32")
    y, err = product64(x, w, b, True)
    z = act64(y, "quick_gelu") + r.double()
    out16 = torch.full((rows, n), float("nan"), dtype=torch.float16, device=eng.device)
    tol = 1.13 * err + 2.0 ** -20 * y.abs() + 2.0 ** -23 * z.abs()
    assert_within(eng.linear(x, w, out16, bias=b, act="quick_gelu", residual=r), z, rounded(z, tol, out16.dtype), "fp16")
    eng.ctx.check()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [1, 40, 200, 400])
def test_linear_activations_and_residual_in_place(eng, act, rows):
    import torch
    rnd, x, w = inputs(eng, 7, rows, 512, 300)
    w = w * 8  # arguments on both flat sides of the activations
    b, r = rnd(300), rnd(rows, 300)
    y, err = product64(x, w, b, True)
    z = act64(y, act) + r.double()
    tol = 1.13 * err + 2.0 ** -20 * y.abs() + 2.0 ** -22 * (z.abs() + r.double().abs())
    out = r.clone()
    assert_within(eng.linear(x, w, out, bias=b, act=act, residual=out), z, rounded(z, tol, out.dtype), act)
    eng.ctx.check()


@pytest.mark.parametrize("rows,k,n,act,bias", [
    (1, 2560, 1280, "silu", False), (1, 8, 1, "gelu", True), (2, 64, 64, "silu", False), (16, 896, 4864, "silu", False),
    (17, 264, 130, "gelu_tanh", True), (40, 1024, 257, "gelu", True), (64, 2560, 2048, "silu", False),
    (77, 2304, 1215, "gelu_tanh", True), (129, 520, 127, "quick_gelu", False), (300, 2048, 384, "silu", True),
    (513, 1000, 260, "none", True), (1024, 512, 1000, "silu", False)])
def test_gate_up(eng, rows, k, n, act, bias):
    import torch
    rnd, x, w = inputs(eng, rows * 3 + k + n, rows, k, n)
    u = (rnd(n, k) / math.sqrt(k)).half()
    bg, bu = (0.3 * rnd(n), 0.3 * rnd(n)) if bias else (None, None)
    gate, eg = product64(x, w, bg, False)
    up, eu = product64(x, u, bu, False)
    ref = act64(gate, act) * up
    # The activation's slope is at most 1.13; the product of the two errors is below 2^-10 of either.
    tol = (1.13 * eg + 2.0 ** -20 * gate.abs()) * up.abs() + act64(gate, act).abs() * eu + eg * eu * 2 + 2.0 ** -22 * ref.abs()
    out = torch.full((rows, n), float("nan"), dtype=torch.float16, device=eng.device)
    assert_within(eng.ffnGateUp(x, w, u, out, act=act, b_gate=bg, b_up=bu), ref, rounded(ref, tol, out.dtype), "gate-up")
    eng.ctx.check()


@pytest.mark.parametrize("rows,k,n", [(1, 2560, 1280), (64, 2560, 640), (100, 2048, 300), (300, 1024, 1000)])
def test_repeats_bitwise(eng, rows, k, n):
    """Split tiles are joined in a fixed order, and neighbours of the output stay as they were."""
    import torch
    rnd, x, w = inputs(eng, 3, rows, k, n)
    u = (rnd(n, k) / math.sqrt(k)).half()
    buf = torch.full((rows + 2, n), 7.0, dtype=torch.float16, device=eng.device)
    first = None
    for _ in range(30):
        eng.ffnGateUp(x, w, u, buf[1:-1])
        y = eng.linear(x, w, torch.empty((rows, n), device=eng.device))
        torch.cuda.synchronize()
        now = (buf[1:-1].clone(), y)
        first = first or now
        assert torch.equal(now[0], first[0]) and torch.equal(now[1], first[1])
        assert (buf[0] == 7).all() and (buf[-1] == 7).all()
    eng.ctx.check()


def test_nonfinite_rows_stay_in_their_rows(eng):
    import torch
    rnd, x, w = inputs(eng, 5, 40, 256, 300)
    x[3, 5], x[17, 0] = float("nan"), float("inf")
    w[8, 2] = float("nan")
    out = eng.linear(x, w, torch.empty((40, 300), device=eng.device))
    eng.ctx.check()
    ref = x.double() @ w.double().t()
    assert torch.equal(torch.isfinite(out), torch.isfinite(ref))
    # Past fp16's range the output is infinite, as a cast of the f32 value is.
    big = eng.linear(torch.full((2, 64), 100.0, device=eng.device).half(), torch.full((3, 64), 100.0, device=eng.device).half(),
                     torch.empty((2, 3), dtype=torch.float16, device=eng.device))
    assert torch.isinf(big).all()


def test_zero_rows_and_empty_range(eng):
    import torch
    rnd, x, w = inputs(eng, 5, 4, 64, 32)
    before = eng.ctx.launches
    eng.linear(x[:0], w, torch.empty((0, 32), device=eng.device))
    eng.ffnGateUp(x[:0], w, w, torch.empty((0, 32), dtype=torch.float16, device=eng.device))
    assert eng.ctx.launches == before


def test_large_output_offsets(eng):
    """rows * n beyond 2^31 elements: the last rows are right."""
    import torch
    rows, k, n = 140000, 8, 15400
    rnd, x, w = inputs(eng, 5, rows, k, n)
    out = torch.empty((rows, n), dtype=torch.float16, device=eng.device)
    eng.linear(x, w, out)
    eng.ctx.check()
    for at in (slice(0, 8), slice(rows // 2, rows // 2 + 8), slice(rows - 8, rows)):
        y, err = product64(x[at], w, None, True)
        assert_within(out[at], y, rounded(y, err, out.dtype), str(at))


@pytest.mark.parametrize("rows,d,ff,act,post,one_plus", [
    (1, 896, 4864, "silu", False, False), (9, 512, 1000, "gelu_tanh", True, True), (64, 2560, 2048, "silu", False, False),
    (200, 256, 520, "silu", False, False), (600, 512, 1024, "gelu_tanh", True, True)])
def test_ffn_block(eng, rows, d, ff, act, post, one_plus):
    """out = h + ffn(rmsnorm(h)): the norm's and the hidden rows' fp16 roundings are part of the block."""
    import torch
    rnd, _, wg = inputs(eng, 17, 1, d, ff)
    wu, wd = (rnd(ff, d) / math.sqrt(d)).half(), (rnd(d, ff) / math.sqrt(ff)).half()
    h = 3.0 * rnd(rows, d)
    norm = 0.1 * rnd(d) if one_plus else 1 + 0.1 * rnd(d)
    pn = 0.1 * rnd(d)
    out = torch.full((rows, d), float("nan"), device=eng.device)
    eng.ffn(h, wg, wu, wd, out, ffn_norm=norm, eps=1e-6, one_plus=one_plus, act=act, post_norm=pn if post else None)
    eng.ctx.check()

    def rms(v, gain):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * (1 + gain.double() if one_plus else gain.double())

    x = rms(h.double(), norm)
    gate, up = x @ wg.double().t(), x @ wu.double().t()
    hid = act64(gate, act) * up
    y = hid @ wd.double().t()
    ref = h.double() + (rms(y, pn) if post else y)
    # Roundings of x and of the hidden rows, 2^-11 of each element, in random directions: the sums'
    # standard deviation is 2^-11 / sqrt(3) of their own size, for gate, up and hidden together at
    # most 2.2 times that; six of them, and the norm keeps relative errors.
    size = y.pow(2).mean(-1, keepdim=True).sqrt()
    tol = 6 * 2.2 * 2.0 ** -11 / math.sqrt(3) * (size * (rms(y, pn).abs().amax() / y.abs().amax() if post else 1.0)) + 2.0 ** -22 * ref.abs() + 1e-5
    assert_within(out, ref, tol, "ffn")


def test_captured_graphs_and_streams(eng):
    """Products captured without a call before, replayed on two streams beside an eager one."""
    import torch
    from brimkern_b200.engine import AttentionEngine
    e = AttentionEngine(0)
    rnd, x, w = inputs(e, 19, 48, 2560, 640)
    u = (rnd(640, 2560) / 50).half()
    xs = [x, x.flip(0).contiguous(), (x * 0.5)]
    outs = [torch.zeros((48, 640), dtype=torch.float16, device=e.device) for _ in xs]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in xs]
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            e.ffnGateUp(xs[i], w, u, outs[i])
        graphs.append(gr)
    want = [e.ffnGateUp(v, w, u, torch.empty_like(outs[0])) for v in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        e.ffnGateUp(xs[2], w, u, outs[2], stream=streams[2])
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert torch.equal(o, v)
    e.ctx.check()
    del graphs
    e.close()


def test_layer_over_shared_prefix(eng):
    """A run of them as a decode step uses them: q / k / v projections, append and attention over the
    shared prefix (fp16 output), the output projection as a linear with the residual, the
    feed-forward block -- against the same layer in 64 bits."""
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache
    rnd, _, _ = inputs(eng, 23, 1, 8, 1)
    dev, B, d, ff, Hq, Hkv, D, P = eng.device, 6, 512, 1024, 8, 4, 64, 150
    W = lambda n, k: (rnd(n, k) / math.sqrt(k)).half()  # noqa: E731
    wq, wk, wv, wo = W(Hq * D, d), W(Hkv * D, d), W(Hkv * D, d), W(d, Hq * D)
    wg, wu, wd = W(ff, d), W(ff, d), W(d, ff)
    gain1, gain2 = 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(d)
    prefix, kv = KvCache(eng.ctx, 1, 1, Hkv, D, P), KvCache(eng.ctx, 1, B, Hkv, D, 4)
    pk, pv = rnd(P, Hkv, D), rnd(P, Hkv, D)
    prefix.write_rows(0, 0, 0, pk, pv)
    cfg = AttnConfig(Hq, Hkv, D, kv_offset=P)
    h = rnd(B, d)
    q, k, v = (torch.empty((B, n), device=dev) for n in (Hq * D, Hkv * D, Hkv * D))
    eng.projQkv(h, wq, wk, wv, q, k, v, attn_norm=gain1)
    att = torch.empty((B, 1, Hq, D), dtype=torch.float16, device=dev)
    eng.stepPrefix(prefix, P, kv, 0, cfg, q.view(B, 1, Hq, D), k.view(B, 1, Hkv, D), v.view(B, 1, Hkv, D), [P] * B, out=att)
    mid = eng.linear(att.view(B, Hq * D), wo, torch.empty((B, d), device=dev), residual=h)
    out = eng.ffn(mid, wg, wu, wd, torch.empty((B, d), device=dev), ffn_norm=gain2)
    eng.ctx.check()

    def rms(t, gain):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * gain.double()

    h64 = h.double()
    n1 = rms(h64, gain1)
    q64, k64, v64 = (n1 @ m.double().t() for m in (wq, wk, wv))
    K = torch.cat([pk.half().double().expand(B, P, Hkv, D), k64.view(B, 1, Hkv, D)], 1)
    V = torch.cat([pv.half().double().expand(B, P, Hkv, D), v64.view(B, 1, Hkv, D)], 1)
    p = torch.softmax(torch.einsum("bhgd,bnhd->bhgn", q64.view(B, Hkv, Hq // Hkv, D), K) / math.sqrt(D), -1)
    a64 = torch.einsum("bhgn,bnhd->bhgd", p, V).reshape(B, Hq * D)
    m64 = h64 + a64 @ wo.double().t()
    x = rms(m64, gain2)
    ref = m64 + (act64(x @ wg.double().t(), "silu") * (x @ wu.double().t())) @ wd.double().t()
    # The framework's tolerance for O(1) outputs: the fp16 roundings (2^-11) of n1, q, p, the attention
    # output, x and the hidden rows, each carried on at a gain of about one.
    assert ((out.double() - ref).abs() <= 2e-3 + 1e-2 * ref.abs()).all(), (out.double() - ref).abs().max().item()


def test_refusals(eng):
    import torch
    from brimkern_b200 import BrkError
    rnd, x, w = inputs(eng, 29, 4, 64, 32)
    out = torch.empty((4, 32), device=eng.device)
    h16 = torch.empty((4, 32), dtype=torch.float16, device=eng.device)
    wide = torch.empty(4 * 64 + 1, dtype=torch.float16, device=eng.device)
    before = eng.ctx.launches
    for bad in (lambda: eng.linear(x.float(), w, out), lambda: eng.linear(x, w.float(), out),
                lambda: eng.linear(x[:, :60].contiguous(), w[:, :60].contiguous(), out),
                lambda: eng.linear(x, w[:, :56].contiguous(), out), lambda: eng.linear(x[:, ::2], w[:, :32].contiguous(), out),
                lambda: eng.linear(x, w, out[:3]), lambda: eng.linear(x, w, out.double()), lambda: eng.linear(x, w, out.cpu()),
                lambda: eng.linear(x, w, out, act="tanh"), lambda: eng.linear(x, w, out, bias=torch.zeros(31, device=eng.device)),
                lambda: eng.linear(x, w, out, residual=h16), lambda: eng.linear(x[0], w, out),
                lambda: eng.linear(wide[1:].view(4, 64), w, out),
                lambda: eng.linear(x, w, out.view(-1)), lambda: eng.linear(x, x, x[:, :4]),
                lambda: eng.ffnGateUp(x, w, w[:31], h16), lambda: eng.ffnGateUp(x, w, w, out),
                lambda: eng.ffn(out, w, w, w, out)):
        with pytest.raises(BrkError):
            bad()
    # Overlapping outputs.
    buf = torch.zeros(4 * 64, dtype=torch.float16, device=eng.device)
    with pytest.raises(BrkError):
        eng.linear(buf.view(4, 64), w, buf[128:].view(4, 32))
    r = torch.zeros(4 * 32 + 4, device=eng.device)
    with pytest.raises(BrkError):
        eng.linear(x, w, r[:-4].view(4, 32), residual=r[4:].view(4, 32))
    wd, hh = torch.zeros((64, 32), dtype=torch.float16, device=eng.device), torch.zeros((4, 64), device=eng.device)
    with pytest.raises(BrkError):
        eng.ffn(hh, w, w, wd, hh)
    assert eng.ctx.launches == before
    eng.linear(x, w, out)
    eng.ctx.check()
