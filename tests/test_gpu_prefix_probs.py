"""The probabilities of decode over a shared prefix carry more than the 11 bits of one fp16 term: a few keys
take all of the softmax, so that nothing averages their roundings out.

K and q have one element that is not zero, so a score is a single product (exact in f32) times the scale.
What is left of the error, relative to sum p |v|: the exponential's argument (2^-24 of at most 20, at each of
exponential, split join and final join: together below 4e-6), ex2 (2^-22), P's two terms (2^-22), the sums
(a few 2^-24): below 2^-17 = 7.6e-6.  One fp16 term alone is off by up to 2.4e-4."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,P,B", [
    (32, 8, 128, 2111, 5),    # the prefix apart, four copies of the query rows
    (32, 8, 128, 1000, 16),   # two copies
    (32, 8, 128, 700, 64),    # two row tiles
    (14, 2, 64, 1100, 64),
    (8, 4, 256, 2113, 8),
    (8, 4, 256, 1025, 70),
    (32, 8, 64, 300, 3),      # one launch
])
def test_few_keys(eng, Hq, Hkv, D, P, B, q8):
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache
    dev = eng.device
    g = torch.Generator(device=dev).manual_seed(P + B)
    prefix, kv = KvCache(eng.ctx, 1, 1, Hkv, D, P, q8=q8), KvCache(eng.ctx, 1, B, Hkv, D, 2, q8=q8)
    k = torch.zeros((P, Hkv, D), device=dev)
    k[:, :, 0] = -3.0
    hot = [1, P // 2, P - 2]  # they lie in different splits, streams and copies
    k[hot, :, 0] = torch.rand((len(hot), Hkv), generator=g, device=dev)
    v = torch.rand((P, Hkv, D), generator=g, device=dev) + 0.1
    prefix.write_rows(0, 0, 0, k, v)
    for b in range(B):
        ko = torch.zeros((1, Hkv, D), device=dev)
        ko[:, :, 0] = torch.rand((1, Hkv), generator=g, device=dev)
        kv.write_rows(0, b, 0, ko, torch.rand((1, Hkv, D), generator=g, device=dev) + 0.1)
    q = torch.zeros((B, 1, Hq, D), device=dev)
    q[..., 0] = 3.0 + 2.0 * torch.rand((B, 1, Hq), generator=g, device=dev)
    q = q.half()
    out = torch.full(q.shape, float("nan"), device=dev)
    cfg = AttnConfig(Hq, Hkv, D, kv_offset=P, scale=1.0)
    eng.decodePrefix(prefix, P, kv, 0, cfg, q, out, [P] * B)
    eng.ctx.check()

    def rows(c, seq, n):
        if c.q8:
            kc, ks, vc, vs = c.read_codes(0, seq, 0, n)
            return kc.double() * ks.double().unsqueeze(-1), vc.double() * vs.double().unsqueeze(-1)
        return tuple(x.double() for x in c.read_rows(0, seq, 0, n))

    pk, pv = rows(prefix, 0, P)
    for b in range(B):
        ok, ov = rows(kv, b, 1)
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[b, 0].double().view(Hkv, Hq // Hkv, D), torch.cat([pk, ok])), -1)
        ref = torch.einsum("hgn,nhd->hgd", p, torch.cat([pv, ov])).reshape(Hq, D)
        err = (out[b, 0].double() - ref).abs() / ref
        assert err.max().item() <= 2.0 ** -17, (b, err.max().item())


@pytest.mark.parametrize("Hq,Hkv,D,P,B,T", [(32, 8, 128, 131072, 512, 1), (8, 4, 256, 70000, 512, 1),
                                            (21, 3, 64, 131072, 441, 4)])  # one split just fills the GPU
def test_long_prefix_and_many_rows(eng, Hq, Hkv, D, P, B, T):
    """Values of one sign: a tensor-core sum loses up to half a step (2^-24) of itself with each of the two
    products of 16 keys (P's terms), so a split may not be long even when many rows fill the GPU with few:
    2048 products of 16384 keys, 1.2e-4."""
    import torch
    from brimkern_b200.engine import AttnConfig, KvCache
    dev = eng.device
    g = torch.Generator(device=dev).manual_seed(P + D)
    prefix, kv = KvCache(eng.ctx, 1, 1, Hkv, D, P), KvCache(eng.ctx, 1, B, Hkv, D, T)
    for c in range(0, P, 16384):
        n = min(16384, P - c)
        prefix.write_rows(0, 0, c, 0.1 * torch.randn((n, Hkv, D), generator=g, device=dev),
                          1 + torch.rand((n, Hkv, D), generator=g, device=dev))
    for b in range(B):
        kv.write_rows(0, b, 0, torch.zeros((T, Hkv, D), device=dev), torch.ones((T, Hkv, D), device=dev))
    q = torch.randn((B, T, Hq, D), generator=g, device=dev).half()
    out = torch.empty(q.shape, device=dev)
    eng.decodePrefix(prefix, P, kv, 0, AttnConfig(Hq, Hkv, D, kv_offset=P), q, out, [P] * B)
    eng.ctx.check()
    k, v = prefix.read_rows(0, 0, 0, P)
    G = Hq // Hkv
    for b, h in ((0, 0), (B // 2, Hkv - 1), (B - 1, 0)):
        heads = slice(h * G, (h + 1) * G)
        z = q[b, 0, heads].double() @ k[:, h].double().t() * D ** -0.5
        p = torch.softmax(torch.cat([z, z.new_zeros((G, 1))], 1), -1)
        ref = p @ torch.cat([v[:, h].double(), v.new_ones((1, D)).double()])
        assert abs(((out[b, 0, heads].double() - ref) / ref).mean().item()) <= 2048 * 2.0 ** -24
