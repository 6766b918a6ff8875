"""Counters of attention over the 4-bit cache: what they take, and captured calls that find some or none."""
import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
D = 128


def setup(lens=(600, 33, 257), n_kv=2, G=4, cap=600):
    from gaac_amd import FP4KVCache
    require_gpu()
    c = FP4KVCache(len(lens), n_kv, cap)
    g = torch.Generator().manual_seed(1)
    for i, L in enumerate(lens): c.prefill(i, *(torch.randn(L, n_kv, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2)))
    q = torch.randn(len(lens), n_kv * G, D, generator=g).to(torch.bfloat16).cuda()
    return c, q, torch.arange(len(lens), dtype=torch.int32, device="cuda")


def capture(f):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g): out = f()
    return g, out


def replayed(g, out, want):
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_counters_are_of_the_calls_and_not_of_the_slots():
    """A cache of many slots that small batches attend over keeps counters for these batches."""
    from gaac_amd import FP4KVCache
    require_gpu()
    c = FP4KVCache(200, 8, 64)
    q, slots = torch.ones(2, 32, D, dtype=torch.bfloat16, device="cuda"), torch.tensor([7, 150], dtype=torch.int32, device="cuda")
    for _ in range(3): c.attention(q, slots, 0.1, nsplit=2)
    held = sum(t.untyped_storage().nbytes() for t in c._tickets.values()) + sum({t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in c._ready}.values())
    assert held <= (1 + 16) * 2 * 8 * 128 and c._captured == 0
    c.attention(q, slots, 0.1)
    assert FP4KVCache(2, 2, 64).attention(q[:, :4], slots - 150, 0.1).shape == (2, 4, D)      # no splits: none


def test_a_call_captured_before_any_other():
    """No call outside of a capture has made counters: the splits are added up by a launch of their own."""
    c, q, slots = setup()
    g, out = capture(lambda: c.attention(q, slots, D ** -0.5, nsplit=4))
    assert c._captured == 0
    replayed(g, out, c.attention(q, slots, D ** -0.5, nsplit=4))


def test_captured_calls_of_more_rows_and_of_fewer():
    """Counters grow with the rows of the calls outside; captured calls that have some keep theirs."""
    c, q, slots = setup()
    one = (q[:1].contiguous(), slots[:1].contiguous())
    want = c.attention(*one, D ** -0.5, nsplit=4)
    graphs = [(*capture(lambda: c.attention(*one, D ** -0.5, nsplit=4)), want)]
    all_rows = lambda: c.attention(q, slots, D ** -0.5, nsplit=4)
    g, out = capture(all_rows)      # more rows than any call before
    assert c._captured == 1
    want = all_rows()
    graphs += [(g, out, want), (*capture(all_rows), want)]
    assert c._captured == 2
    for _ in range(3):
        for x in graphs: replayed(*x)
        assert torch.equal(all_rows(), want)


def test_a_busy_stream_does_not_keep_a_graph_from_its_counters():
    """Counters made by a call on a stream that has much to do are zero for a graph on another stream at once."""
    c, q, slots = setup()
    call = lambda: c.attention(q, slots, D ** -0.5, nsplit=4)
    want = call()
    c._no_counters()
    torch.cuda.synchronize()
    busy = torch.cuda.Stream()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(20_000_000)
        late = call()
    assert len(c._ready) == 16 and all(int(s.cpu().abs().max()) == 0 for s in c._ready)
    torch.cuda.synchronize()
    assert torch.equal(late, want)
    replayed(*capture(call), want)


def test_a_captured_call_takes_one_set(monkeypatch):
    """Also where the binding leaves the call to Python (strided or misaligned queries, slots with gaps, a whole number as scale), and none where it is refused."""
    from gaac_amd import _lib
    c, q, slots = setup()
    x = torch.zeros(3, 16, D, dtype=torch.bfloat16, device="cuda")
    x[:, ::2] = q
    odd = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    gaps = torch.stack([slots, slots + 5], 1)[:, 0]
    calls = [lambda: c.attention(q, slots, D ** -0.5, nsplit=4), lambda: c.attention(x[:, ::2], slots, D ** -0.5, nsplit=4), lambda: c.attention(odd, slots, D ** -0.5, nsplit=4),
             lambda: c.attention(q, gaps, D ** -0.5, nsplit=4), lambda: c.attention(q, slots, 1, nsplit=4)]
    want = [f() for f in calls]
    for w in want[1:4]: assert torch.equal(w, want[0])
    for python in (False, True):
        if python: monkeypatch.setattr(_lib, "_calls", _lib._CtypesCalls())
        for f, w in zip(calls, want):
            before = c._captured
            g, out = capture(f)
            assert c._captured == before + 1
            replayed(g, out, w)
        before = c._captured
        def refused():
            with pytest.raises(RuntimeError, match="GQA group size"): c.attention(q[:, :3], slots, D ** -0.5, nsplit=4)
            with pytest.raises(RuntimeError, match="slots int32"): c.attention(q, slots[:2], D ** -0.5, nsplit=4)
            return q.clone()
        capture(refused)
        assert c._captured == before and len({s.data_ptr() for s in c._ready + c._given}) == len(c._ready + c._given)


def test_threads_that_capture_at_once_get_sets_of_their_own():
    """The sets are taken one by one: many threads that take counters as captured calls do never hold the same."""
    import threading
    c, q, slots = setup()
    c.attention(q, slots, D ** -0.5, nsplit=4)
    start, took = threading.Barrier(8), []
    real = torch._C._cuda_isCurrentStreamCapturing
    torch._C._cuda_isCurrentStreamCapturing = lambda: True
    try:
        def take():
            start.wait()
            for _ in range(2): took.append(c._counters(6))
        threads = [threading.Thread(target=take) for _ in range(8)]
        for t in threads: t.start()
        for t in threads: t.join()
    finally: torch._C._cuda_isCurrentStreamCapturing = real
    assert len({t.data_ptr() for t in took}) == 16 and c._captured == 16 and c._ready == []


def test_counters_of_dropped_graphs_are_taken_again():
    from gaac_amd import fp4_cache
    c, q, slots = setup()
    call = lambda: c.attention(q, slots, D ** -0.5, nsplit=4)
    want = call()
    kept = capture(call)
    for i in range(fp4_cache.CAPTURES + 10):
        with c.captured_counters() as counters: g, out = capture(call)
        assert len(counters) == 1 and c._captured == 2
        if i % 10 == 0:
            replayed(g, out, want)
            replayed(*kept, want)
        torch.cuda.synchronize()
        del g, out
        c.give_back(counters)
        assert c._captured == 1
    with pytest.raises(RuntimeError, match="give_back expects counters"): c.give_back(counters)
    with c.captured_counters() as counters:
        call()      # not captured: none
        capture(lambda: [pytest.raises(RuntimeError, c.attention, q, slots[:2], D ** -0.5, nsplit=4), q.clone()][1])      # refused: none
    assert counters == [] and c._captured == 1
    many = (q.repeat(4, 1, 1), slots.repeat(4))
    with c.captured_counters() as counters: capture(call)
    c.attention(*many, D ** -0.5, nsplit=2)      # larger sets are wanted from here on
    c.give_back(counters)
    assert all(s.numel() >= 12 * 2 * 32 for s in c._ready)


def test_the_decode_loop_captures_anew_as_often_as_it_likes():
    from gaac_amd import fp4_cache
    from gaac_amd.serving import DecodeRunner, ModelConfig, Weights
    dev = require_gpu()
    cfg = ModelConfig(hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, ffn=512, vocab=500, rope_theta=10000.0, max_len=2500)
    run = DecodeRunner(Weights(cfg, dev, seed=1), n_slots=2, kv="fp4")
    for i in range(2): run.prefill(i, torch.randint(0, cfg.vocab, (1900 + i,), generator=torch.Generator(device=dev).manual_seed(2 + i), device=dev))
    for i in range(fp4_cache.CAPTURES + 3):
        run.start_decode(torch.tensor([5, 6], device=dev))
        assert [c._captured for c in run.caches] == [1, 1]      # with splits, and counters for them
        if i % 20 == 0: run.decode(2)
    held = run.lens.tolist()
    graph = run.decode(3)
    run.start_decode(torch.tensor([5, 6], device=dev), use_graph=False)
    assert [c._captured for c in run.caches] == [0, 0] and held[1] == held[0] + 1 and graph.shape == (3, 2)


def test_counters_of_many_caches_come_from_one_stretch_of_memory():
    """40 layers that each make their first counters reserve what these take, not a stretch of the allocator's for each."""
    from gaac_amd import FP4KVCache
    require_gpu()
    caches = [FP4KVCache(1, 2, 64) for _ in range(40)]
    q, slots = torch.ones(1, 8, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    caches[0].attention(q, slots, 0.1, nsplit=2)
    before = torch.cuda.memory_reserved()
    for c in caches[1:]: c.attention(q, slots, 0.1, nsplit=2)
    assert torch.cuda.memory_reserved() - before <= 4 << 20 and len({c._ready[0].data_ptr() for c in caches}) == 40
