"""GPU tests of ``tp_cache_evict`` (``PagedKVCache.evict_slots`` / ``evict``):
moves and comparisons alone, so everything is equal to the restatement."""

import math

import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cache(lengths, hk, dim, page, maxp, dtype=torch.float16, seed=0, ordered=False):
    from turbopress_b200.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, P, cap = len(lengths), len(lengths) * maxp + 1, maxp * page
    kp, vp = (torch.randn(P, hk, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    table = torch.randperm(P, generator=g, device=DEV)[:B * maxp].reshape(B, maxp).int().contiguous()
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    scores = torch.rand(B, hk, cap, generator=g, device=DEV)
    live = torch.arange(cap, device=DEV) < lens[:, None, None]
    order = torch.rand(B, hk, cap, generator=g, device=DEV)
    if ordered:
        order = torch.arange(cap, device=DEV).expand(B, hk, cap).float()
    places = order.masked_fill(~live, 2.0 + cap).argsort(-1).argsort(-1)
    places = torch.where(live, places, -1).int()
    cache = PagedKVCache.from_tensors(kp, vp, table, lens, scores=scores, positions=places,
                                      next_pos=lens.clamp(min=0))
    return cache, g


def _check(cache, budget, recent=0, sinks=0):
    ref = R.evict(cache.k_pages[0], cache.v_pages[0], cache.block_table, cache.lengths, cache.next_pos, cache.scores[0],
                  cache.positions[0], budget, recent, sinks)
    was = [t.clone() for t in (cache.lengths, cache.scores, cache.positions, cache.next_pos)]
    lengths, scores, positions = cache.evict_slots(budget, recent=recent, sinks=sinks)
    assert torch.equal(lengths, ref[2])
    assert torch.equal(positions, ref[4])
    assert torch.equal(scores.view(torch.int32), ref[3].view(torch.int32))
    assert torch.equal(cache.k_pages[0], ref[0]) and torch.equal(cache.v_pages[0], ref[1])
    for a, b in zip(was, (cache.lengths, cache.scores, cache.positions, cache.next_pos)):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    return lengths, scores, positions


@pytest.mark.parametrize("hk,dim,page,dtype", [(2, 64, 16, torch.float16), (1, 128, 8, torch.bfloat16), (3, 80, 4, torch.float16),
                                               (2, 256, 1, torch.bfloat16), (1, 8, 32, torch.float16)])
@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (1, 1, 0), (16, 4, 4), (31, 0, 31), (33, 33, 0), (64, 10, 2), (200, 7, 0)])
def test_evict(hk, dim, page, dtype, budget, recent, sinks):
    maxp = -(-200 // page)
    cache, _ = _cache([200, 17, 64, 0, 65, -1, 1, 33, 199], hk, dim, page, maxp, dtype, seed=budget + dim)
    _check(cache, budget, recent, sinks)


@pytest.mark.parametrize("budget", [5, 40, 99])
def test_equal_scores_keep_the_lower_slots(budget):
    cache, g = _cache([100, 90], 2, 64, 16, 7, seed=3)
    cache.scores.fill_(0.25)
    _check(cache, budget)
    cache.scores[:, :, :, ::3] = 0.5
    _check(cache, budget, recent=3)
    cache.scores.copy_(torch.randint(0, 4, cache.scores.shape, generator=g, device=DEV).float())
    _check(cache, budget, recent=5, sinks=2 if budget > 6 else 0)


def test_scores_at_the_type_s_ends():
    """NaN above all, infinities, both zeros equal, negative and subnormal scores."""
    cache, g = _cache([120], 4, 64, 16, 8, seed=4)
    vals = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-40, -1e-40, 1.0, -1.0, 3e38, -3e38], device=DEV)
    cache.scores.copy_(vals[torch.randint(0, len(vals), cache.scores.shape, generator=g, device=DEV)])
    for budget in (3, 20, 57, 100, 119):
        _check(cache, budget)
        _check(cache, budget, recent=3)


def test_long_caches():
    """More slots than threads, an odd budget, whole heads tied."""
    cache, g = _cache([5001, 4096, 3000], 2, 16, 16, 313, seed=5)
    _check(cache, 1023, recent=100, sinks=4)
    cache.scores[0, 0, 0] = 0.0
    _check(cache, 2047)


@pytest.mark.parametrize("slots,budget,tied", [(50_000, 3001, False), (50_000, 40_000, True), (40_960, 20_479, True)])
def test_caches_past_the_shared_memory(slots, budget, tied):
    """Keys formed anew in each pass (above 40960 slots), more words than threads, many equal scores."""
    cache, g = _cache([slots, slots - 12_345], 1, 8, 32, -(-slots // 32), seed=12)
    if tied:
        cache.scores.copy_(torch.randint(0, 3, cache.scores.shape, generator=g, device=DEV).float())
    _check(cache, budget, recent=64, sinks=4)


@pytest.mark.parametrize("slots", [203, 2051, 4098])
def test_capacities_of_odd_size(slots):
    """Pages of one slot: rows of scores and positions that are not 16-byte aligned."""
    cache, _ = _cache([slots, slots - 1, slots // 2], 2, 16, 1, slots, seed=slots)
    for budget in (50, slots // 2 + 1, slots - 2):
        _check(cache, budget, recent=7, sinks=2)


def test_budget_past_the_capacity_or_the_lengths():
    cache, _ = _cache([64, 3], 2, 64, 16, 4, seed=6)
    for budget in (64, 65, 1000):
        lengths, scores, positions = _check(cache, budget)
        assert torch.equal(lengths, cache.lengths) and torch.equal(positions, cache.positions[0])
    cache.lengths[0] = 1 << 30  # past the capacity: cut to it
    _check(cache, 20)


def test_missing_pages_are_left_out():
    cache, _ = _cache([100, 100], 2, 64, 16, 7, seed=7)
    cache.block_table[0, 5] = -1
    cache.block_table[0, 1] = cache.num_pages + 3
    _check(cache, 50)


def test_the_same_call_again_gives_the_same():
    """Sources lie above the budget and destinations below it: a repeated call moves the same rows."""
    cache, _ = _cache([150], 2, 64, 16, 10, seed=8)
    a = _check(cache, 60)
    k = cache.k_pages.clone()
    b = cache.evict_slots(60)
    assert torch.equal(cache.k_pages, k) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_attention_does_not_see_the_difference():
    """Evicting slots that carry no weight leaves the attention over the kept ones."""
    cache, g = _cache([90, 70], 2, 64, 16, 7, seed=9)
    q = torch.randn(2, 1, 4, 64, generator=g, device=DEV).half()
    B, hk, cap = cache.scores.shape[1:]
    cache.lengths.sub_(1)  # the last slot is the step's token
    full = cache.attend(q, accumulate=False)
    ref, _, w = R.attention(q, cache.k_pages[0], cache.v_pages[0], cache.block_table, cache.lengths)
    cache.lengths.add_(1)
    for budget in (60, 40):
        keep = w.float()
        cache.scores[0].copy_(keep)
        new_len, scores, positions = cache.evict_slots(budget)
        cache.lengths.copy_(new_len - 1)
        got = cache.attend(q)
        for b in range(B):
            for h in range(hk):
                assert abs(float(scores[b, h].sum()) - float(keep[b, h].topk(budget).values.sum())) < 1e-5
        err = float((got.double() - ref).abs().max())
        lost = 1 - float((scores.sum(-1) / keep.sum(-1)).min())
        assert err <= 2 * lost * 2 * float(cache.v_pages.abs().max()) + 2e-3
        cache.lengths.copy_(new_len)
        w = torch.where(torch.arange(cap, device=DEV) < budget, R.attention(
            q, cache.k_pages[0], cache.v_pages[0], cache.block_table, new_len - 1)[2], 0.0)
    assert full.shape == got.shape


def test_evict_all_layers():
    from turbopress_b200.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(10)
    cache = PagedKVCache(2, 2, 64, 16, 16, 8, layers=3, track_weights=True)
    cache.block_table.copy_(torch.randperm(16, generator=g, device=DEV).reshape(2, 8))
    for t in (cache.k_pages, cache.v_pages):
        t.normal_(generator=g)
    cache.scores.uniform_(generator=g)
    cache.positions.copy_(torch.arange(128, device=DEV))
    cache.lengths.copy_(torch.tensor([128, 50], dtype=torch.int32))
    cache.next_pos.copy_(cache.lengths)
    ref = [R.evict(cache.k_pages[i], cache.v_pages[i], cache.block_table, cache.lengths, cache.next_pos, cache.scores[i],
                   cache.positions[i], 60, 8, 2) for i in range(3)]
    cache.evict(60, recent=8, sinks=2)
    for i in range(3):
        assert torch.equal(cache.k_pages[i], ref[i][0]) and torch.equal(cache.v_pages[i], ref[i][1])
        assert torch.equal(cache.scores[i], ref[i][3]) and torch.equal(cache.positions[i], ref[i][4])
    assert cache.lengths.tolist() == [60, 50] and cache.next_pos.tolist() == [128, 50]


def test_graph_and_stream():
    cache, _ = _cache([150, 20], 2, 64, 16, 10, seed=11)
    ref = R.evict(cache.k_pages[0], cache.v_pages[0], cache.block_table, cache.lengths, cache.next_pos, cache.scores[0],
                  cache.positions[0], 60)
    cache._evict_ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        new = cache.evict_slots(60)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(new[1], ref[3]) and torch.equal(cache.k_pages[0], ref[0])


def test_refusals():
    from turbopress_b200 import _abi
    from turbopress_b200.paged import PagedKVCache
    cache, _ = _cache([20], 1, 64, 16, 2)
    for bad in (dict(budget=0), dict(budget=4, recent=5), dict(budget=4, sinks=-1), dict(budget=4, recent=2, sinks=3),
                dict(budget=4, recent=-1), dict(budget=4, layer=1)):
        with pytest.raises(ValueError):
            cache.evict_slots(**bad)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 64, 2, 16, 2).evict_slots(4)
    big = PagedKVCache(1, 1, 8, 1, 1 << 20, 2, track_weights=True)
    with pytest.raises(RuntimeError):  # more slots than the selection's bit map holds
        big.evict_slots(4)
    assert _abi.lib().tp_cache_evict(None, None, None, 0, None) == _abi.TP_ERR_ARG
