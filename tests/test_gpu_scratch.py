"""The scratch of the shared-prefix and linear operators: it belongs to a stream or to a captured graph, and
goes (to later captures, or back to the device) when that is gone."""
import gc
import time

import pytest

pytestmark = pytest.mark.gpu

Hq, Hkv, D, B = 32, 8, 128, 20


def _setup(P):
    import torch
    from brimkern_b200.engine import AttentionEngine, AttnConfig, KvCache
    e = AttentionEngine(0)
    g = torch.Generator(device=e.device).manual_seed(P)
    rnd = lambda *s: torch.randn(s, generator=g, device=e.device)  # noqa: E731
    prefix, kv = KvCache(e.ctx, 1, 1, Hkv, D, P, q8=True), KvCache(e.ctx, 1, B, Hkv, D, 8, q8=True)
    prefix.write_rows(0, 0, 0, rnd(P, Hkv, D), rnd(P, Hkv, D))
    for b in range(B):
        kv.write_rows(0, b, 0, rnd(4, Hkv, D), rnd(4, Hkv, D))
    q = rnd(B, 1, Hq, D).half()
    cfg = lambda p: AttnConfig(Hq, Hkv, D, kv_offset=p)  # noqa: E731

    def close():
        prefix.close()
        kv.close()
        e.close()
    return e, lambda out, p=P, **kw: e.decodePrefix(prefix, p, kv, 0, cfg(p), q, out, [p + 3] * B, **kw), q, close


def _free(device):
    import torch
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info(device)[0]


def _capture(call, out, **kw):
    import torch
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        call(out, **kw)
    return gr


def test_captures_that_are_gone_hold_no_memory():
    import torch
    P = 6000
    e, call, q, close = _setup(P)
    out, want = torch.zeros_like(q), call(torch.empty_like(q)).clone()
    one = 2 * Hkv * P * D * 2  # the staged codes of one call: what a capture holds at least
    for i in range(40):
        if i == 5:
            before = _free(e.device)
        gr = _capture(call, out)
        if i % 8 == 0:
            out.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del gr
        time.sleep(0.002)  # CUDA says that a graph is gone on a thread of its own
    assert before - _free(e.device) < 4 * one
    # Lengths that grow from capture to capture: what is outgrown goes too.
    before = _free(e.device)
    for p in range(1000, P, 250):
        gr = _capture(call, out, p=p)
        del gr
        time.sleep(0.002)
    assert before - _free(e.device) < 4 * one
    e.ctx.check()
    close()


def test_graphs_take_over_scratch_but_share_none():
    """Two live graphs replayed at once beside a third that took over a dead one's scratch; and a graph that
    needs more than the dead one had."""
    import torch
    e, call, q, close = _setup(6000)
    outs = [torch.zeros_like(q) for _ in range(3)]
    want = [call(torch.empty_like(q), p=p).clone() for p in (5000, 6000, 1200)]
    a, dead = _capture(call, outs[0], p=5000), _capture(call, torch.empty_like(q), p=2000)
    dead.replay()
    torch.cuda.synchronize()
    del dead
    gc.collect()
    time.sleep(0.05)
    b, c = _capture(call, outs[1], p=6000), _capture(call, outs[2], p=1200)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, gr in zip(streams, (a, b, c)):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    e.ctx.check()
    close()
    del a, b, c  # after the context: what CUDA then says about their scratch finds it closed
    gc.collect()
    time.sleep(0.05)


def test_call_within_a_capture_that_needs_more():
    """The nodes captured before keep the buffer that the later call of the same capture outgrows."""
    import torch
    e, call, q, close = _setup(6000)
    outs = [torch.zeros_like(q) for _ in range(3)]
    sizes = (1100, 6000, 3000)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        for o, p in zip(outs, sizes):
            call(o, p=p)
    want = [call(torch.empty_like(q), p=p).clone() for p in sizes]
    for _ in range(5):
        for o in outs:
            o.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    e.ctx.check()
    close()


def test_streams_that_are_gone_hold_no_memory():
    """Far more streams than keep their scratch, each with a call in flight when the next ones come."""
    import torch
    runtime = pytest.importorskip("cuda.bindings.runtime")
    P = 3000
    e, call, q, close = _setup(P)
    want = call(torch.empty_like(q)).clone()
    one = 2 * Hkv * P * D * 2
    outs = [torch.zeros_like(q) for _ in range(200)]
    torch.cuda.synchronize()
    before = _free(e.device)
    for i, o in enumerate(outs):
        err, s = runtime.cudaStreamCreateWithFlags(runtime.cudaStreamNonBlocking)
        assert int(err) == 0
        call(o, stream=torch.cuda.ExternalStream(int(s)))
        if i % 2:
            runtime.cudaStreamSynchronize(s)
        assert int(runtime.cudaStreamDestroy(s)[0]) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert before - _free(e.device) < 70 * one * 1.25
    e.ctx.check()
    # The first stream's scratch may be gone; it gets another.
    assert torch.equal(call(torch.empty_like(q)), want)
    close()


def test_growing_calls_of_one_stream():
    import torch
    e, call, q, close = _setup(6000)
    sizes = [1000, 1500, 2500, 4000, 6000, 2000]
    got = [call(torch.empty_like(q), p=p) for p in sizes]  # queued back to back
    torch.cuda.synchronize()
    for o, p in zip(got, sizes):
        assert torch.equal(o, call(torch.empty_like(q), p=p))
    x, w = torch.randn((300, 2560), device=e.device).half(), torch.randn((2560, 2560), device=e.device).half()
    y = e.linear(x, w, torch.empty((300, 2560), device=e.device))
    assert torch.equal(y, e.linear(x, w, torch.empty_like(y)))
    e.ctx.check()
    close()


def test_graph_dropped_while_it_runs():
    """Its scratch is nobody else's before its last replay is through."""
    import torch
    e, call, q, close = _setup(6000)
    want = [call(torch.empty_like(q), p=p).clone() for p in (6000, 5900)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(15):
        outs = [torch.zeros_like(q) for _ in range(2)]
        torch.cuda.synchronize()
        gr = _capture(call, outs[0], p=6000)
        with torch.cuda.stream(streams[0]):
            torch.cuda._sleep(5_000_000)
            gr.replay()
        del gr
        gc.collect()
        gr = _capture(call, outs[1], p=5900)
        with torch.cuda.stream(streams[1]):
            for _ in range(20):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        del gr
    e.ctx.check()
    close()


def test_stream_grows_while_another_captures():
    """A call outside the capture, on a stream of its own, allocates and frees meanwhile."""
    import torch
    e, call, q, close = _setup(6000)
    side = torch.cuda.Stream()
    outs = [torch.zeros_like(q) for _ in range(4)]
    sizes = (1100, 2000, 6000, 3000)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        call(outs[0], p=sizes[0])
        call(outs[1], p=sizes[1], stream=side)
        call(outs[2], p=sizes[2], stream=side)
        call(outs[3], p=sizes[3])
    gr.replay()
    torch.cuda.synchronize()
    for o, p in zip(outs, sizes):
        assert torch.equal(o, call(torch.empty_like(q), p=p))
    e.ctx.check()
    close()
