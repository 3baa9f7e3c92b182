"""Decode over a shared prefix with int8 rows whose V is far from one in size: the V scales enter the
probabilities before these are rounded to fp16, so their size must not cost bits.  f32 outputs against 64
bits, at the relative tolerance that N(0,1) rows meet (tests/test_gpu_prefix.py) and no absolute one."""
import math

import pytest

pytestmark = pytest.mark.gpu

REL = 2.0 ** -11 + 1.1e-4


def _sizes(kind, n, g, dev):
    """The size of each row's V."""
    import torch
    if kind == "mixed":  # neighbouring rows three orders of magnitude apart
        return torch.where(torch.arange(n, device=dev) % 2 == 0, 1e-3, 1.0)
    if kind == "zeros":  # every third row is zero (its scale is the quantiser's smallest)
        return torch.where(torch.arange(n, device=dev) % 3 == 0, 0.0, 1e-3)
    if kind == "growing":  # the size grows along the keys
        return torch.logspace(-4, 2, n, device=dev)
    if kind == "falling":
        return torch.logspace(2, -4, n, device=dev)
    return torch.full((n,), float(kind), device=dev)


KINDS = ["1", "1e-2", "1e-3", "1e-4", "1e-8", "1e3", "1e7", "1e20", "mixed", "zeros", "growing", "falling"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hkv,D,P,own,T,q8p,q8o,kw", [
    (8, 8, 64, 0, [900, 64], 1, True, True, {}),                                      # own rows alone
    (32, 8, 128, 300, [5, 130], 1, True, True, {}),                                   # one launch
    (32, 8, 128, 1003, [1 + 20 * i for i in range(17)], 1, True, True, {}),           # apart, four copies of the rows
    (8, 4, 256, 667, [1 + i for i in range(40)], 1, True, True, dict(softcap=50.0)),  # apart, two copies, head 256
    (32, 8, 64, 1100, [4 + i for i in range(40)], 4, True, True, dict(window=900)),   # apart, row tiles
    (32, 8, 128, 1003, [1 + 20 * i for i in range(17)], 1, True, False, {}),          # int8 prefix, fp16 own rows
    (32, 8, 128, 2111, [3, 1, 65, 500, 7], 1, False, True, {}),                       # the reverse
])
def test_v_of_any_size(eng, kind, Hq, Hkv, D, P, own, T, q8p, q8o, kw):
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache
    dev = eng.device
    g = torch.Generator(device=dev).manual_seed(77 + P)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    cfg = AttnConfig(Hq, Hkv, D, kv_offset=P, **kw)
    caches = []
    for q8, lens in ((q8p, [P] if P else []), (q8o, own)):
        if not lens:
            caches.append(None)
            continue
        kv = KvCache(eng.ctx, 1, len(lens), Hkv, D, max(lens) + 3, q8=q8)
        for b, n in enumerate(lens):
            size = _sizes(kind, n, g, dev) if q8 else torch.full((n,), min(6e4 / 6, max(1e-3, float(_sizes(kind, n, g, dev).max()))), device=dev)
            kv.write_rows(0, b, 0, rnd(n, Hkv, D), rnd(n, Hkv, D) * size.view(n, 1, 1))
        caches.append(kv)
    prefix, kv = caches
    q = rnd(len(own), T, Hq, D).half()
    out = torch.full(q.shape, float("nan"), device=dev)
    past = [P + n - T for n in own]
    eng.decodePrefix(prefix, P, kv, 0, cfg, q, out, past)
    eng.ctx.check()

    def rows(c, seq, n):
        if c.q8:
            kc, ks, vc, vs = c.read_codes(0, seq, 0, n)
            return kc.double() * ks.double().unsqueeze(-1), vc.double() * vs.double().unsqueeze(-1)
        return tuple(x.double() for x in c.read_rows(0, seq, 0, n))

    scale, G = 1 / math.sqrt(D), Hq // Hkv
    for b, n in enumerate(own):
        k, v = rows(kv, b, n)
        if P:
            pk, pv = rows(prefix, 0, P)
            k, v = torch.cat([pk, k]), torch.cat([pv, v])
        for t in range(T):
            end = past[b] + t + 1
            lo = max(0, end - cfg.window) if cfg.window else 0
            z = torch.einsum("hgd,nhd->hgn", q[b, t].double().view(Hkv, G, D), k[lo:end]) * scale
            if cfg.softcap:
                z = cfg.softcap * torch.tanh(z / cfg.softcap)
            p = torch.softmax(z, -1)
            ref = torch.einsum("hgn,nhd->hgd", p, v[lo:end]).reshape(Hq, D)
            mag = torch.einsum("hgn,nhd->hgd", p, v[lo:end].abs()).reshape(Hq, D)
            err = (out[b, t].double() - ref).abs()
            bad = ~(err <= REL * mag)
            assert not bad.any(), (b, t, int(bad.sum()), (err / (REL * mag)).max().item())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 1e30])
@pytest.mark.parametrize("P,own,W", [(8001, [3, 30, 301, 5, 6, 7], 7007), (3001, [2, 3, 4, 9], 2502), (301, [5, 9], 251)])
def test_scales_below_every_window(eng, bad, P, own, W):
    """Rows before the first attended one may hold anything, though loads round down to a multiple of four."""
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache
    dev = eng.device
    g = torch.Generator(device=dev).manual_seed(P)
    Hq, Hkv, D, B = 32, 8, 128, len(own)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    prefix, kv = KvCache(eng.ctx, 1, 1, Hkv, D, P, q8=True), KvCache(eng.ctx, 1, B, Hkv, D, max(own), q8=True)
    prefix.write_rows(0, 0, 0, rnd(P, Hkv, D), rnd(P, Hkv, D))
    for b, n in enumerate(own):
        kv.write_rows(0, b, 0, rnd(n, Hkv, D), rnd(n, Hkv, D))
    cfg = AttnConfig(Hq, Hkv, D, kv_offset=P, window=W)
    q, past = rnd(B, 1, Hq, D).half(), [P + n - 1 for n in own]
    first = min(past) - W + 1
    assert first % 4 and first < P
    want = eng.decodePrefix(prefix, P, kv, 0, cfg, q, torch.empty_like(q), past)
    kc, ks, vc, vs = prefix.read_codes(0, 0, 0, first)
    prefix.write_codes(0, 0, 0, kc, torch.full_like(ks, bad), vc, torch.full_like(vs, bad))
    got = eng.decodePrefix(prefix, P, kv, 0, cfg, q, torch.empty_like(q), past)
    eng.ctx.check()
    assert torch.isfinite(want).all() and torch.equal(got, want)
