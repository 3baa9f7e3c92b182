"""Windows that fill the ring's stages to the last key, over caches with a few more rows than the window: the
first attended row is then no multiple of four, to which int8 caches round their first load down, and the
newest rows -- here one that takes nearly all of the softmax -- are in the last split's last stage.
Against 64 bits over the rows the caches hold; the tolerance is the framework's own for O(1) outputs."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _reference(k, v, q, cfg, end):
    import torch
    G = cfg.n_heads // cfg.n_kv_heads
    lo = max(0, end - cfg.window)
    z = torch.einsum("hgd,nhd->hgn", q.double().view(cfg.n_kv_heads, G, cfg.head_dim), k[lo:end]) / math.sqrt(cfg.head_dim)
    return torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), v[lo:end]).reshape(cfg.n_heads, cfg.head_dim)


def _rows64(kv, seq, n):
    if kv.q8:
        kc, ks, vc, vs = kv.read_codes(0, seq, 0, n)
        return kc.double() * ks.double().unsqueeze(-1), vc.double() * vs.double().unsqueeze(-1)
    k, v = kv.read_rows(0, seq, 0, n)
    return k.double(), v.double()


def _inputs(eng, g, Hq, Hkv, D, T, own, q8):
    """Caches whose newest T rows point along the queries, 4 standard deviations of score above the rest."""
    import torch
    from brimkern_b200.engine import KvCache
    rnd = lambda *s: torch.randn(s, generator=g, device=eng.device)  # noqa: E731
    q = (rnd(1, 1, 1, D) + 0.1 * rnd(len(own), T, Hq, D)).half()
    kv = KvCache(eng.ctx, 1, len(own), Hkv, D, max(own) + 5, q8=q8)
    for b, n in enumerate(own):
        k, v = rnd(n, Hkv, D), rnd(n, Hkv, D)
        k[n - T:] = 1.5 * q[b, :, :1].float()
        v[n - T:] += 5.0
        kv.write_rows(0, b, 0, k, v)
    return q, kv


CASES = [(D, W, over, T) for D, W in ((128, 64), (128, 128), (128, 512), (64, 256), (256, 32), (256, 64))
         for over, T in ((1, 1), (2, 1), (3, 1), (3, 2), (5, 4))]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("D,W,over,T", CASES)
def test_decode(eng, D, W, over, T, q8):
    import torch
    from brimkern_b200.engine import AttnConfig
    g = torch.Generator(device=eng.device).manual_seed(D + W + over)
    Hq, Hkv = 16, 2
    own = [W + over, 3 + T, W + T]
    q, kv = _inputs(eng, g, Hq, Hkv, D, T, own, q8)
    cfg = AttnConfig(Hq, Hkv, D, window=W)
    past = [n - T for n in own]
    out = eng.recAttention(kv, 0, cfg, q.float(), torch.empty(q.shape, device=eng.device), past, "decode")
    eng.ctx.check()
    for b, n in enumerate(own):
        k, v = _rows64(kv, b, n)
        for t in range(T):
            ref = _reference(k, v, q[b, t], cfg, past[b] + t + 1)
            assert ((out[b, t].double() - ref).abs() <= 2e-3 + 1e-2 * ref.abs()).all(), (b, t)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("P,D,W,over,T,batch", [(P,) + c + (3,) for P in (36, 37) for c in CASES] + [
    # Only some sequences see the prefix: its own kernel and, beside it, the own rows' splits.
    (5000, 128, 4096, 1, 1, 16), (5000, 128, 4096, 2, 1, 16), (5000, 128, 4096, 3, 1, 16), (5000, 128, 4096, 3, 2, 16)])
def test_decode_prefix(eng, P, D, W, over, T, batch, q8):
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache
    g = torch.Generator(device=eng.device).manual_seed(D + W + over)
    Hq, Hkv = 32, 8
    own = [W + over, W + T, W + over + 1] + [1 + T] * (batch - 3)
    q, kv = _inputs(eng, g, Hq, Hkv, D, T, own, q8)
    prefix = KvCache(eng.ctx, 1, 1, Hkv, D, P, q8=q8)
    prefix.write_rows(0, 0, 0, torch.randn((P, Hkv, D), generator=g, device=eng.device),
                      torch.randn((P, Hkv, D), generator=g, device=eng.device))
    cfg = AttnConfig(Hq, Hkv, D, window=W, kv_offset=P)
    past = [P + n - T for n in own]
    pk, pv = _rows64(prefix, 0, P)
    out = eng.decodePrefix(prefix, P, kv, 0, cfg, q, torch.empty_like(q), past)
    eng.ctx.check()
    for b, n in enumerate(own):
        k, v = _rows64(kv, b, n)
        k, v = torch.cat([pk, k]), torch.cat([pv, v])
        for t in range(T):
            ref = _reference(k, v, q[b, t], cfg, past[b] + t + 1)
            assert ((out[b, t].double() - ref).abs() <= 2e-3 + 1e-2 * ref.abs()).all(), (b, t)
