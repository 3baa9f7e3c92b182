"""Decode attention over a shared prefix (brk_attn_decode_prefix / brk_attn_step_prefix) against the
softmax in 64 bits over the rows the caches hold.

Tolerance, from the kernels' roundings, relative to sum_j p_j |v_j| of the output (p the softmax):
the probabilities are rounded to fp16 (half a step 2^-11 = 4.9e-4); a score is a sum of D / 16
tensor-core steps, each truncated by at most 2^-22 of sum |q k| (at D 256, scale 1/16 and N(0,1) rows:
16 * 2.4e-7 * 10.2 = 4e-5), the softcap's tanh is off by a few 1e-7 absolute times c log2(e) = 72
(3e-5), the exponential by 2^-22: together below 1.1e-4.  int8 codes enter the products exactly and
their scales multiply f32 scores and probabilities: nothing is added.  An fp16 output adds half a
step of its own, 2^-11 |o|."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _cfg(Hq, Hkv, D, P, **kw):
    from brimkern_b200.engine import AttnConfig
    return AttnConfig(Hq, Hkv, D, kv_offset=P, **kw)


def _rows(kv, seq, n, layer=0):
    """The n first rows of a sequence as the cache holds them, in 64 bits: K, V [n, Hkv, D]."""
    if kv.q8:
        kc, ks, vc, vs = kv.read_codes(layer, seq, 0, n)
        return kc.double() * ks.double().unsqueeze(-1), vc.double() * vs.double().unsqueeze(-1)
    k, v = kv.read_rows(layer, seq, 0, n)
    return k.double(), v.double()


def _check(prefix, pseq, P, kv, cfg, q, out, past, layer=0):
    import torch
    torch.cuda.synchronize()
    B, T, Hq, D = q.shape
    Hkv, G = cfg.n_kv_heads, cfg.n_heads // cfg.n_kv_heads
    scale = cfg.scale or 1.0 / math.sqrt(D)
    pk, pv = _rows(prefix, pseq, P, layer) if P else (torch.zeros((0, Hkv, D), dtype=torch.float64, device=q.device),) * 2
    q64 = q.half().double()  # the tensor cores' operand
    rel = 2.0 ** -11 + 1.1e-4
    for b in range(B):
        ok, ov = _rows(kv, b, past[b] + T - P, layer)
        k, v = torch.cat([pk, ok]), torch.cat([pv, ov])
        for t in range(T):
            end = past[b] + t + 1
            lo = max(0, end - cfg.window) if cfg.window else 0
            z = torch.einsum("hgd,nhd->hgn", q64[b, t].view(Hkv, G, D), k[lo:end]) * scale
            if cfg.softcap:
                z = cfg.softcap * torch.tanh(z / cfg.softcap)
            p = torch.softmax(z, -1)
            ref = torch.einsum("hgn,nhd->hgd", p, v[lo:end]).reshape(Hq, D)
            mag = torch.einsum("hgn,nhd->hgd", p, v[lo:end].abs()).reshape(Hq, D)
            err = (out[b, t].double() - ref).abs()
            tol = rel * mag + (2.0 ** -11 * ref.abs() + 2.0 ** -25 if out.dtype == torch.float16 else 0.0) + 1e-6
            bad = ~(err <= tol)
            assert not bad.any(), (f"sequence {b} token {t}: {int(bad.sum())} of {bad.numel()} outside, worst "
                                   f"{(err / tol).max().item():.3g} of the tolerance")


def _fill(eng, g, Hkv, D, P, own, q8p, q8o, pseqs=1, layers=1, spare=3):
    """Prefix cache (P rows in its last sequence) and own caches (own[b] rows), N(0,1)."""
    import torch
    from brimkern_b200.engine import KvCache
    dev = eng.device
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    prefix = KvCache(eng.ctx, layers, pseqs, Hkv, D, P + spare, q8=q8p) if P else None
    kv = KvCache(eng.ctx, layers, len(own), Hkv, D, max(own) + spare, q8=q8o)
    for layer in range(layers):
        if P:
            prefix.write_rows(layer, pseqs - 1, 0, rnd(P, Hkv, D), rnd(P, Hkv, D))
        for b, n in enumerate(own):
            if n:
                kv.write_rows(layer, b, 0, rnd(n, Hkv, D), rnd(n, Hkv, D))
    return prefix, kv


CASES = [
    # name, Hq, Hkv, D, P, own rows per sequence (new tokens included), T, prefix int8, own int8, q, out, kwargs
    ("one", 8, 8, 64, 1, [1], 1, False, False, "f16", "f16", {}),
    ("no_prefix", 14, 2, 64, 0, [5, 1, 70], 1, False, False, "f16", "f32", {}),
    ("p63", 14, 2, 64, 63, [5, 1, 70, 33], 1, False, False, "f16", "f16", {}),
    ("p64", 14, 2, 64, 64, [64, 65, 1, 2], 1, False, False, "f32", "f32", {}),
    ("p65", 32, 8, 128, 65, [3] * 5, 1, False, False, "f16", "f16", {}),
    ("p130_t3", 32, 8, 128, 130, [3, 4, 100], 3, False, False, "f32", "f16", {}),
    ("rows128", 32, 8, 128, 300, list(range(1, 33)), 1, False, False, "f16", "f16", {}),
    ("rows132", 32, 8, 128, 321, list(range(1, 34)), 1, False, False, "f16", "f16", {}),
    ("rows256", 32, 8, 128, 1000, [1 + 7 * i for i in range(64)], 1, False, False, "f16", "f16", {}),
    ("rows300", 32, 8, 128, 777, [1 + i for i in range(75)], 1, False, False, "f16", "f32", {}),
    ("d64_long", 32, 8, 64, 9001, [1, 250, 17], 1, False, False, "f16", "f16", {}),
    ("d64_rows448", 14, 2, 64, 500, [2 + i for i in range(64)], 1, False, False, "f16", "f16", {}),
    ("d256", 8, 4, 256, 500, [1, 2, 300, 64], 1, False, False, "f16", "f16", {}),
    ("d256_rows130", 8, 4, 256, 259, [1 + 3 * i for i in range(65)], 1, False, False, "f16", "f32", {}),
    ("d256_cap", 8, 4, 256, 1025, [1 + 5 * i for i in range(32)], 1, False, False, "f32", "f16",
     dict(softcap=50.0, scale=1 / 16)),
    ("window_in_own", 32, 8, 128, 200, [90, 100, 80], 1, False, False, "f16", "f16", dict(window=50)),
    ("window_1", 32, 8, 128, 200, [1, 2], 1, False, False, "f16", "f16", dict(window=1)),
    ("window_ragged", 32, 8, 128, 1000, [2, 40, 300, 301], 2, False, False, "f16", "f16", dict(window=300)),
    ("window_d256_cap", 8, 4, 256, 700, [5, 200, 33], 1, False, False, "f16", "f16", dict(window=256, softcap=30.0)),
    ("window_all", 32, 8, 64, 130, [5, 7], 1, False, False, "f16", "f16", dict(window=10 ** 6)),
    ("q8_both", 32, 8, 128, 1003, [1, 77, 300], 1, True, True, "f16", "f16", {}),
    ("q8_both_t2", 32, 8, 128, 515, [2 + i for i in range(17)], 2, True, True, "f16", "f16", {}),
    ("q8_prefix_only", 14, 2, 64, 259, [1, 77, 300, 4], 1, True, False, "f32", "f16", {}),
    ("q8_own_only", 8, 4, 256, 259, [1, 77, 300, 4], 1, False, True, "f16", "f16", {}),
    ("q8_window", 32, 8, 64, 1001, [3, 30, 301], 1, True, True, "f16", "f32", dict(window=307)),
    ("q8_d256_cap", 8, 4, 256, 333, [1 + i for i in range(40)], 1, True, True, "f16", "f16", dict(softcap=50.0)),
    ("mha", 8, 8, 128, 150, [9, 10], 4, False, False, "f16", "f16", {}),
    ("g64", 64, 1, 64, 150, [9, 10], 1, False, False, "f16", "f16", {}),
    ("split_own", 8, 8, 128, 100, [5000, 3], 1, False, False, "f16", "f16", {}),
    ("tiny_scale", 32, 8, 128, 150, [9, 10], 1, False, False, "f16", "f16", dict(scale=1e-4)),
    # A prefix of few bytes a unit is read by the own rows' kernel itself; here with its rows split over
    # clusters and over more splits than a cluster takes, with two row tiles, and with splits that hold
    # prefix rows only, own rows only, or both.
    ("split_prefix", 14, 2, 64, 8190, [3], 1, False, False, "f16", "f16", {}),
    ("split_mixed", 14, 2, 64, 1000, [3, 900, 64], 1, False, False, "f32", "f32", {}),
    ("split_t5", 32, 8, 128, 700, [5, 333], 5, False, False, "f16", "f16", {}),
    ("split_window", 8, 2, 128, 3000, [5, 333, 40], 2, False, False, "f16", "f32", dict(window=1500)),
    ("split_q8", 8, 1, 256, 3001, [5, 333], 1, True, True, "f16", "f16", dict(softcap=30.0)),
    # More bytes than that: a kernel of its own reads the prefix once.
    ("apart", 32, 8, 128, 2111, [3, 1, 65, 500, 7], 1, False, False, "f16", "f16", {}),
    ("apart_t3", 32, 8, 128, 2177, [3, 4, 100, 20], 3, False, False, "f32", "f16", {}),
    ("apart_d64", 14, 2, 64, 1100, [2 + i for i in range(64)], 1, False, False, "f16", "f16", {}),
    ("apart_d256", 8, 4, 256, 2113, [1, 2, 300, 64], 1, False, False, "f16", "f32", {}),
    ("apart_window", 32, 8, 128, 5000, [2, 40, 300, 301], 2, False, False, "f16", "f16", dict(window=4500)),
    ("apart_window_cap", 8, 4, 256, 4000, [5, 200, 33, 1], 1, False, False, "f16", "f16", dict(window=2500, softcap=30.0)),
    ("apart_q8", 32, 8, 128, 1003, [1 + 20 * i for i in range(17)], 1, True, True, "f16", "f16", {}),
    ("apart_q8_t2", 32, 8, 128, 1030, [2 + i for i in range(17)], 2, True, True, "f32", "f16", {}),
    ("apart_q8_window", 32, 8, 64, 8001, [3, 30, 301, 5, 6, 7], 1, True, True, "f16", "f32", dict(window=7007)),
    ("apart_q8_cap", 8, 4, 256, 667, [1 + i for i in range(40)], 1, True, True, "f16", "f16", dict(softcap=50.0)),
    ("apart_mha", 8, 8, 128, 4200, [9, 10], 4, False, False, "f16", "f16", {}),
    ("apart_g64", 64, 1, 64, 9001, [9 + i for i in range(8)], 1, False, False, "f16", "f16", {}),
    ("apart_split_own", 8, 8, 128, 4200, [5000, 3], 1, False, False, "f16", "f16", {}),
]


@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_decode_prefix(eng, case):
    import torch
    name, Hq, Hkv, D, P, own, T, q8p, q8o, qt, ot, kw = case
    g = torch.Generator(device=eng.device).manual_seed(len(name) * 131 + P)
    prefix, kv = _fill(eng, g, Hkv, D, P, own, q8p, q8o)
    cfg = _cfg(Hq, Hkv, D, P, **kw)
    B = len(own)
    q = torch.randn((B, T, Hq, D), generator=g, device=eng.device)
    if qt == "f16":
        q = q.half()
    out = torch.full((B, T, Hq, D), float("nan"), dtype=torch.float16 if ot == "f16" else torch.float32, device=eng.device)
    past = [P + n - T for n in own]
    for _ in range(2):  # twice: the scratch's counters are back at zero
        eng.decodePrefix(prefix, P, kv, 0, cfg, q, out, past)
        eng.ctx.check()
        _check(prefix, 0, P, kv, cfg, q, out, past)


@pytest.mark.parametrize("P", [100, 2800])
def test_other_sequence_and_layer_and_stale_rows(eng, P):
    """The named prefix sequence and layer are read, and rows behind the prefix's length or a
    sequence's last position -- NaN, as a rewound or foreign cache may hold -- are not."""
    import torch
    g = torch.Generator(device=eng.device).manual_seed(5)
    Hq, Hkv, D, own = 32, 8, 128, [7, 70, 65]
    prefix, kv = _fill(eng, g, Hkv, D, P, own, False, False, pseqs=3, layers=2, spare=40)
    nan = torch.full((40, Hkv, D), float("nan"), device=eng.device)
    for layer in range(2):
        prefix.write_rows(layer, 2, P, nan, nan)
        for b, n in enumerate(own):
            room = max(own) + 40 - n
            kv.write_rows(layer, b, n, nan[:room], nan[:room])
    cfg = _cfg(Hq, Hkv, D, P)
    q = torch.randn((3, 1, Hq, D), generator=g, device=eng.device).half()
    past = [P + n - 1 for n in own]
    for layer in (1, 0):
        out = torch.empty_like(q)
        eng.decodePrefix(prefix, P, kv, layer, cfg, q, out, past, prefix_seq=2)
        eng.ctx.check()
        _check(prefix, 2, P, kv, cfg, q, out, past, layer)


@pytest.mark.parametrize("B", [8, 40])
@pytest.mark.parametrize("mag", [1.0, 6.0])
def test_sharp_scores(eng, mag, B):
    """Scores whose maximum grows late and differently from row to row (the running maximum and the
    rescale), with one key that takes everything."""
    import torch
    g = torch.Generator(device=eng.device).manual_seed(9)
    Hq, Hkv, D, P, own = 32, 8, 128, 640, [3] * B
    prefix, kv = _fill(eng, g, Hkv, D, P, own, False, False)
    ramp = torch.linspace(0.05, mag, P, device=eng.device).view(P, 1, 1)
    prefix.write_rows(0, 0, 0, torch.randn((P, Hkv, D), generator=g, device=eng.device) * ramp,
                      torch.randn((P, Hkv, D), generator=g, device=eng.device))
    cfg = _cfg(Hq, Hkv, D, P)
    q = (torch.randn((B, 1, Hq, D), generator=g, device=eng.device) * 2).half()
    out = torch.empty_like(q)
    past = [P + 2] * B
    eng.decodePrefix(prefix, P, kv, 0, cfg, q, out, past)
    eng.ctx.check()
    # Larger scores: the truncation bound of the module's text scales with sum |q k| (2 mag).
    torch.cuda.synchronize()
    pk, pv = _rows(prefix, 0, P)
    for b in range(B):
        ok, ov = _rows(kv, b, 3)
        k, v = torch.cat([pk, ok]), torch.cat([pv, ov])
        z = torch.einsum("hgd,nhd->hgn", q[b, 0].double().view(Hkv, 4, D), k) / math.sqrt(D)
        za = torch.einsum("hgd,nhd->hgn", q[b, 0].double().abs().view(Hkv, 4, D), k.abs()) / math.sqrt(D)
        p = torch.softmax(z, -1)
        ref = torch.einsum("hgn,nhd->hgd", p, v)
        # p_j is off by the score's error e_j and the sum's; both at most max_j e_j.
        ej = 8 * 2.0 ** -22 * za + 2.0 ** -23 * z.abs() * 3
        rel = 2.0 ** -11 + 2.0 ** -21
        tol = torch.einsum("hgn,nhd->hgd", p * (rel + 2 * ej.amax(-1, keepdim=True)), v.abs()) + 2.0 ** -11 * ref.abs() + 2.0 ** -24
        err = (out[b, 0].double().view(Hkv, 4, D) - ref).abs()
        assert (err <= tol).all(), (err / tol).max().item()


@pytest.mark.parametrize("P", [2000, 2100])
def test_repeated_calls_are_bitwise_equal(eng, P):
    """The same call gives the same bits every time (ordered merges)."""
    import torch
    g = torch.Generator(device=eng.device).manual_seed(11)
    Hq, Hkv, D, own = 32, 8, 128, [1500, 20, 700, 1]
    prefix, kv = _fill(eng, g, Hkv, D, P, own, False, False)
    cfg = _cfg(Hq, Hkv, D, P)
    q = torch.randn((4, 1, Hq, D), generator=g, device=eng.device).half()
    past = [P + n - 1 for n in own]
    outs = [eng.decodePrefix(prefix, P, kv, 0, cfg, q, torch.empty_like(q), past) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("P", [333, 1700])
def test_step_prefix_chain(eng, P):
    """Append + attention, step after step: equal to attention over one cache that holds prefix and
    own rows (brk_attn_step), and the appended rows are brk_attn_append's bits."""
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache, RopeTable
    g = torch.Generator(device=eng.device).manual_seed(21)
    dev = eng.device
    Hq, Hkv, D, B, steps = 32, 8, 128, 5, 6
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    rope = RopeTable(eng.ctx, D, 1e6, None, P + steps)
    qn, kn = 1 + 0.02 * rnd(D), 1 + 0.02 * rnd(D)
    pk, pv = rnd(P, Hkv, D), rnd(P, Hkv, D)
    prefix, own = KvCache(eng.ctx, 1, 1, Hkv, D, P), KvCache(eng.ctx, 1, B, Hkv, D, steps)
    whole = KvCache(eng.ctx, 1, B, Hkv, D, P + steps)
    prefix.write_rows(0, 0, 0, pk, pv)
    for b in range(B):
        whole.write_rows(0, b, 0, pk, pv)
    cfg = AttnConfig(Hq, Hkv, D, q_norm=qn, k_norm=kn, rope=rope, kv_offset=P)
    plain = AttnConfig(Hq, Hkv, D, q_norm=qn, k_norm=kn, rope=rope)
    for i in range(steps):
        q, k, v = rnd(B, 1, Hq, D), rnd(B, 1, Hkv, D), rnd(B, 1, Hkv, D)
        past = [P + i] * B
        got = eng.stepPrefix(prefix, P, own, 0, cfg, q, k, v, past)
        ref = eng.attentionLayer(whole, 0, plain, q, k, v, past)
        eng.ctx.check()
        # Both round q and the probabilities to fp16, in another order: each is within 2^-11 + 1.1e-4
        # of sum p |v| (< 1.2 here, 338 N(0,1) rows or more and their softmax) from the exact result.
        assert (got - ref).abs().max().item() <= 2 * (2.0 ** -11 + 1.1e-4 + 2.0 ** -11) * 1.2
        for b in range(B):
            a, c = own.read_rows(0, b, i, 1), whole.read_rows(0, b, P + i, 1)
            assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
        half = torch.empty((B, 1, Hq, D), dtype=torch.float16, device=dev)
        eng.decodePrefix(prefix, P, own, 0, cfg, eng.appendKv(own, 0, cfg, q, k, v, torch.empty_like(q), past), half, past)
        eng.ctx.check()
        assert torch.equal(half, got.half())


@pytest.mark.parametrize("P", [700, 3000])
def test_captured_graphs_and_streams(eng, P):
    """Two captured graphs and an eager call share no scratch: replayed at once on three streams, each
    gives what it gives alone; the capture needs no call before it."""
    import torch
    from brimkern_b200.engine import AttentionEngine
    e = AttentionEngine(0)  # a context that has run nothing
    g = torch.Generator(device=e.device).manual_seed(31)
    Hq, Hkv, D = 32, 8, 128
    own = [1500, 20, 700, 1]
    prefix, kv = _fill(e, g, Hkv, D, P, own, False, False)
    cfg = _cfg(Hq, Hkv, D, P)
    past = [P + n - 1 for n in own]
    qs = [torch.randn((4, 1, Hq, D), generator=g, device=e.device).half() for _ in range(3)]
    outs = [torch.zeros_like(q) for q in qs]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            e.decodePrefix(prefix, P, kv, 0, cfg, qs[i], outs[i], past)
        graphs.append(gr)
    want = [e.decodePrefix(prefix, P, kv, 0, cfg, q, torch.empty_like(q), past) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        e.decodePrefix(prefix, P, kv, 0, cfg, qs[2], outs[2], past, stream=streams[2])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    e.ctx.check()
    del graphs
    prefix.close()
    kv.close()
    e.close()


def test_branches_of_one_graph(eng):
    """Calls captured on two streams of one capture become branches that may run at once: they share no
    scratch either (prefix splits, split matrix products)."""
    import torch
    g = torch.Generator(device=eng.device).manual_seed(37)
    Hq, Hkv, D, P, own = 32, 8, 128, 4000, [1500, 20, 700, 1]
    prefix, kv = _fill(eng, g, Hkv, D, P, own, False, False)
    cfg = _cfg(Hq, Hkv, D, P)
    past = [P + n - 1 for n in own]
    qs = [torch.randn((4, 1, Hq, D), generator=g, device=eng.device).half() for _ in range(2)]
    x = [torch.randn((600, 2560), generator=g, device=eng.device).half() for _ in range(2)]
    w = torch.randn((2560, 2560), generator=g, device=eng.device).half()
    outs, ys = [torch.zeros_like(q) for q in qs], [torch.zeros_like(t) for t in x]

    def work(i):
        for _ in range(4):
            eng.decodePrefix(prefix, P, kv, 0, cfg, qs[i], outs[i], past)
            eng.linear(x[i], w, ys[i])
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(2):
        work(i)
    torch.cuda.synchronize()
    want = [t.clone() for t in outs + ys]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=main):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            work(1)
        work(0)
        main.wait_stream(side)
    for _ in range(20):
        for t in outs + ys:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, v) for t, v in zip(outs + ys, want))
    eng.ctx.check()


def test_refusals(eng):
    """Calls the operator does not cover raise and launch nothing."""
    import torch
    from brimkern_b200 import BrkError
    from brimkern_b200.engine import AttentionEngine
    g = torch.Generator(device=eng.device).manual_seed(41)
    Hq, Hkv, D, P, own = 32, 8, 128, 100, [4, 9]
    prefix, kv = _fill(eng, g, Hkv, D, P, own, False, False)
    cfg = _cfg(Hq, Hkv, D, P)
    q = torch.randn((2, 1, Hq, D), generator=g, device=eng.device).half()
    past = [P + n - 1 for n in own]
    other, other_kv = _fill(eng, g, 4, D, P, own, False, False)
    e2 = AttentionEngine(0)
    foreign, foreign_kv = _fill(e2, g, Hkv, D, P, own, False, False)
    before = eng.ctx.launches
    call = lambda **kw: eng.decodePrefix(*[kw.get(n, d) for n, d in (  # noqa: E731
        ("prefix", prefix), ("prefix_len", P), ("kv", kv), ("layer", 0), ("cfg", cfg), ("q", q),
        ("out", torch.empty_like(q)), ("past", past))], prefix_seq=kw.get("prefix_seq", 0))
    for bad in (dict(prefix=None), dict(prefix=other), dict(prefix=foreign), dict(prefix_len=P - 1), dict(prefix_len=-1),
                dict(cfg=_cfg(Hq, Hkv, D, P + 1)), dict(layer=1), dict(prefix_seq=1), dict(prefix_seq=-1),
                dict(prefix_len=P + 4, cfg=_cfg(Hq, Hkv, D, P + 4), past=[P + 8, P + 9]),
                dict(past=[P - 1, P]), dict(past=[P + 12, P]), dict(past=[P]), dict(q=q[:, :, :1].contiguous()),
                dict(q=q.double()), dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), dict(q=q.cpu()), dict(out=q), dict(out=torch.empty_like(q)[:1]),
                dict(out=torch.empty((2, 1, Hq, D), dtype=torch.bfloat16, device=eng.device)),
                dict(q=torch.empty((2, 17, Hq, D), dtype=torch.float16, device=eng.device),
                     out=torch.empty((2, 17, Hq, D), dtype=torch.float16, device=eng.device))):
        with pytest.raises(BrkError):
            call(**bad)
    f = torch.randn((2, 1, Hq, D), device=eng.device)
    kvf = torch.randn((2, 1, Hkv, D), device=eng.device)
    with pytest.raises(BrkError):
        eng.stepPrefix(prefix, P, kv, 0, cfg, f, kvf[:1], kvf, past)
    with pytest.raises(BrkError):
        eng.stepPrefix(prefix, P, prefix, 0, cfg, f[:1].contiguous(), kvf[:1].contiguous(), kvf[:1].contiguous(), [P])
    assert eng.ctx.launches == before
    call()  # the engine still works
    eng.ctx.check()
    for x in (prefix, kv, other, other_kv, foreign, foreign_kv):
        x.close()
    e2.close()
