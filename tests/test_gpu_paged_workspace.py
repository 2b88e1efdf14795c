"""GPU tests of the workspaces that a ``PagedKVCache`` owns: what is outgrown is
given back unless a graph was recorded with it, and such a graph's status is
still read."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cache(batch=4, pages=64, heads=2, dim=64):
    from turbopress_b200.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = PagedKVCache(batch, heads, dim, batch * pages, 16, pages, track_weights=True)
    cache.block_table.copy_(torch.arange(batch * pages, device=DEV).view(batch, pages))
    cache.k_pages.normal_(generator=g)
    cache.v_pages.normal_(generator=g)
    cache.scores.uniform_(generator=g)
    cache.lengths.fill_(500)
    cache.next_pos.fill_(500)
    return cache, g


def _q(g, tokens, heads, batch=4, dim=64):
    return torch.randn(batch, tokens, heads, dim, generator=g, device=DEV).half()


def test_outgrown_workspaces_are_given_back():
    cache, g = _cache()
    sizes = ((1, 2), (2, 16), (8, 16), (32, 16), (200, 16), (500, 64))
    calls = [_q(g, *s) for s in sizes]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    seen = []
    for q in calls:
        cache.attend(q, accumulate=True)
        seen.append(cache._ws.numel())
    assert seen[-1] > 2 * seen[0]
    assert torch.cuda.memory_allocated() - before <= cache._ws.numel() + (1 << 20)
    for budget in (1, 100, 400):
        cache.evict_slots(budget)
    assert torch.cuda.memory_allocated() - before <= cache._ws.numel() + cache._evict_ws.numel() + (1 << 20)


def test_a_stream_that_still_runs_keeps_what_it_uses():
    """Grown on another stream than the workspace was made on: the first one's
    later allocations do not get memory that the second still uses."""
    cache, g = _cache()
    small, large = _q(g, 1, 4), _q(g, 64, 32)
    want = cache.attend(small).clone()
    first = cache._ws.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        got = cache.attend(small)
        size = cache._ws.numel()
        cache.attend(large, accumulate=True)
        end = side.record_event()
    other = torch.full((size,), 255, dtype=torch.uint8, device=DEV)  # (of the size that was just given up)
    assert end.query() or other.data_ptr() != first  # (once the stream has come to its end, it may be reused)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_a_graph_keeps_its_workspaces():
    cache, g = _cache()
    small, large = _q(g, 1, 4), _q(g, 64, 32)
    want = cache.attend(small).clone()
    kept = cache.evict_slots(300)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        held = cache.attend(small)
        cache.attend(small)
        again = cache.evict_slots(300)
    ws, ev = cache._ws, cache._evict_ws
    cache.attend(large, accumulate=True)  # outgrows the graph's workspace
    cache.evict_slots(511)
    assert cache._ws is not ws
    junk = [torch.full((t.numel(),), 255, dtype=torch.uint8, device=DEV) for t in (ws, ev) for _ in range(4)]
    assert all(t.data_ptr() not in (ws.data_ptr(), ev.data_ptr()) for t in junk)
    assert [t is ws for t in cache._captured] == [True]
    cache.k_pages.copy_(cache.k_pages)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again[0], kept[0])
    cache.status()
    ws[2048] = 1  # the record of a wait that gave up in a replay
    with pytest.raises(RuntimeError, match="wait"):
        cache.status()
    cache.status()
    assert held.shape == want.shape
    fresh = cache.attend(small)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, fresh)
    larger = _q(g, 512, 64)
    with pytest.raises(RuntimeError, match="capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            cache.attend(larger, accumulate=True)


def test_rotaries_of_the_past_are_let_go():
    """A cache that meets many Rotary objects holds a few of them, and still takes each as it is."""
    import gc
    import weakref

    from turbopress_b200.rotary import Rotary
    cache, g = _cache()
    q, kv = _q(g, 1, 4), _q(g, 1, 2)
    seen = []
    for i in range(40):
        rotary = Rotary(64, theta=10000.0 + i)
        want, _ = rotary(q, kv, cache.next_pos.long()[:, None])
        assert torch.equal(cache.append(rotary, q, kv, kv), want)
        seen.append(weakref.ref(rotary))
    del rotary
    gc.collect()
    assert sum(r() is not None for r in seen) <= 16


def test_a_cache_keeps_its_tensors():
    """Another tensor in the place of lengths would not reach the kernels: refused; in-place writes count."""
    cache, g = _cache()
    q = _q(g, 1, 4)
    for name in ("lengths", "block_table", "k_pages", "v_pages", "scores", "positions"):
        with pytest.raises(AttributeError, match="write into it"):
            setattr(cache, name, getattr(cache, name).clone())
    long = cache.attend(q)
    cache.lengths -= 400
    short = cache.attend(q)
    assert not torch.equal(long, short)
    cache.lengths[:] = 500
    assert torch.equal(cache.attend(q), long)
    cache.next_pos = torch.full((4,), 77, dtype=torch.int32, device=DEV)  # (read anew by every call)
    kv = _q(g, 1, 2)
    from turbopress_b200.rotary import Rotary
    rotary = Rotary(64)
    want, _ = rotary(q, kv, torch.full((4, 1), 77, device=DEV))
    assert torch.equal(cache.append(rotary, q, kv, kv), want)
