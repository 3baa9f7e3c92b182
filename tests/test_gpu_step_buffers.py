"""The steps' own buffers when they are given a stream that is not the current one: the block that the
kernels on that stream write must not be handed out again to the current stream's work behind them."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", ["stepPrefix", "attentionLayer"])
def test_step_on_another_stream_keeps_its_buffers(eng, entry, monkeypatch):
    import torch
    from brimkern_b200 import _lib as L
    from brimkern_b200.engine import AttnConfig, KvCache
    dev = eng.device
    Hq, Hkv, D, B, P = 32, 8, 128, 3, 70
    g = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    kv = KvCache(eng.ctx, 1, B, Hkv, D, 4)
    q, k, v = rnd(B, 1, Hq, D), rnd(B, 1, Hkv, D), rnd(B, 1, Hkv, D)
    if entry == "stepPrefix":
        prefix = KvCache(eng.ctx, 1, 1, Hkv, D, P)
        prefix.write_rows(0, 0, 0, rnd(P, Hkv, D), rnd(P, Hkv, D))
        name, at = "brk_attn_step_prefix", (13, 14)  # q_work, out
        step = lambda **kw: eng.stepPrefix(prefix, P, kv, 0, AttnConfig(Hq, Hkv, D, kv_offset=P), q, k, v, [P] * B, **kw)  # noqa: E731
    else:
        name, at = "brk_attn_step", (10, 11)
        step = lambda **kw: eng.attentionLayer(kv, 0, AttnConfig(Hq, Hkv, D), q, k, v, [0] * B, **kw)  # noqa: E731
    seen = []
    fn = getattr(L.lib(), name)
    address = lambda a: a if isinstance(a, int) else a.value  # noqa: E731
    monkeypatch.setattr(L.lib(), name, lambda *args: (seen.append([address(args[i]) for i in at]), fn(*args))[1])
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    seen.clear()
    out = step(stream=side)
    other = [torch.empty_like(q) for _ in range(8)]  # the current stream's next allocations of that size
    taken = {t.data_ptr() for t in other}
    assert seen[0][1] == out.data_ptr()
    assert seen[0][0] not in taken and seen[0][1] not in taken
    with torch.cuda.stream(side):  # its own stream may have it again, in order
        assert seen[0][0] in {t.data_ptr() for t in [torch.empty_like(q) for _ in range(64)]}
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    # The output is read on the current stream: dropped there, it is not handed out on the side stream
    # before what the current stream had queued.
    want.add_(1.0)  # (the kernel's first launch, which may wait for the device)
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)
    out.add_(1.0)
    del out
    with torch.cuda.stream(side):
        assert seen[0][1] not in {t.data_ptr() for t in [torch.empty_like(q) for _ in range(8)]}
    torch.cuda.synchronize()
    eng.ctx.check()


def test_step_prefix_refuses_before_it_allocates(eng):
    """On a stream of its own too, inputs of the wrong device or type come back as the library's error."""
    import torch
    from brimkern_b200 import BrkError
    from brimkern_b200.engine import AttnConfig, KvCache
    kv = KvCache(eng.ctx, 1, 2, 2, 64, 4)
    q, k = torch.zeros((2, 1, 4, 64), device=eng.device), torch.zeros((2, 1, 2, 64), device=eng.device)
    before = eng.ctx.launches
    for bad in (q.cpu(), q.half(), q.transpose(2, 3)):
        for stream in (None, torch.cuda.Stream()):
            with pytest.raises(BrkError):
                eng.stepPrefix(None, 0, kv, 0, AttnConfig(4, 2, 64), bad, k, k, [0, 0], stream=stream)
    assert eng.ctx.launches == before
