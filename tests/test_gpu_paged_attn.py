"""GPU tests of ``tp_paged_attn`` (``PagedKVCache.attend``) against a 64-bit
restatement.

Tolerances: a score is a 32-bit sum of up to 256 products, its error below
E = 2^-24 * 16 * sum|q_i k_i| * scale (sums of 16 on the tensor cores, then 16
in sequence), i.e. 1e-5 for sum|q_i k_i| scale < 10 as in all inputs here but
the peaked ones, which give their own; a probability is then within 2 E
relative (score and normaliser), and stays so as two 16-bit terms (2^-16).  So
out is within 4 E max|v| of the exact value before its one rounding (half an
ulp: 2^-11, bf16 2^-8), lse within 2 E, a slot's weight within 4 E of its value
times the rows (plus 1e-7).
"""

import math

import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cache(lengths, T, hk, dim, page, dtype, seed, track=False, token_major=False, garbage=float("nan")):
    """A cache whose unseen slots hold `garbage`; pages in random order."""
    from turbopress_b200.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(seed)
    counts = [max(1, -(-(n + T) // page)) for n in lengths]
    P, maxp = sum(counts) + 2, max(counts) + 1
    shape = (P, page, hk, dim) if token_major else (P, hk, page, dim)
    kp, vp = (torch.full(shape, garbage, device=DEV, dtype=dtype) for _ in range(2))
    if token_major:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    order = torch.randperm(P, generator=g, device=DEV).int()
    table = torch.full((len(lengths), maxp), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        table[b, :c] = order[at:at + c]
        at += c
        s = torch.arange(max(0, n + T) if n >= 0 else 0, device=DEV)
        for x in (kp, vp):
            x[table[b].long()[s // page], :, s % page] = torch.randn(len(s), hk, dim, generator=g, device=DEV).to(dtype)
    scores = torch.rand(len(lengths), hk, maxp * page, generator=g, device=DEV) * 0.01 if track else None
    cache = PagedKVCache.from_tensors(kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scores=scores)
    return cache, g


def _check(cache, q, scale=None, accumulate=False, E=1e-5):
    before = None if cache.scores is None else cache.scores.clone()
    out, lse = cache.attend(q, scale=scale, accumulate=accumulate, return_lse=True)
    kp, vp = cache.k_pages[0], cache.v_pages[0]
    ref, ref_lse, w = R.attention(q, kp, vp, cache.block_table, cache.lengths, scale)
    top = float(torch.nan_to_num(vp.float(), 0, 0, 0).abs().max())
    tol = HALF_ULP[q.dtype] * ref.abs() * (1 + 2.0 ** -6) + 4 * E * top + 2.0 ** -25
    err = (out.double() - ref).abs()
    assert not (~(err <= tol)).any(), float((err / tol).max())
    live = ref_lse > -math.inf
    assert torch.equal(lse > -math.inf, live)
    assert float((lse.double() - ref_lse)[live].abs().amax() if live.any() else 0) <= 2 * E
    if accumulate:
        rows = q.shape[1] * q.shape[2] // cache.kv_heads
        got = cache.scores[0].double() - before[0].double()
        lim = 4 * E * w + 1e-7 * rows + 2.0 ** -23 * cache.scores[0].double().abs()
        assert not (~((got - w).abs() <= lim)).any(), float(((got - w).abs() / lim).max())
    elif before is not None:
        assert torch.equal(before, cache.scores)
    return out


LENGTHS = {"one": [0], "short": [0, 1, 14, 15, 16, 62, 63, 64, 65], "idle": [5, -1, 130, -1], "long": [5000],
           "ragged": [700, 3, 0, 2047, 129, 64]}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("T,hq,hk,dim,page", [(1, 32, 8, 128, 16), (1, 7, 1, 64, 8), (5, 16, 8, 128, 32), (3, 24, 2, 80, 1),
                                              (4, 16, 1, 256, 64), (33, 12, 4, 96, 16), (1, 2, 2, 8, 128), (2, 40, 1, 128, 16)])
def test_attention(T, hq, hk, dim, page, lengths, dtype):
    cache, g = _cache(LENGTHS[lengths], T, hk, dim, page, dtype, T + hq + dim, track=True)
    q = torch.randn(cache.batch, T, hq, dim, generator=g, device=DEV).to(dtype)
    out = _check(cache, q)
    for b, n in enumerate(LENGTHS[lengths]):
        if n < 0:
            assert (out[b] == 0).all()
    _check(cache, q, accumulate=True)
    assert torch.equal(out, cache.attend(q))  # the same bits again: the joins do not depend on timing


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", ["short", "ragged", "idle"])
@pytest.mark.parametrize("T,hq,hk,dim,page", [(3, 16, 2, 128, 16), (5, 10, 2, 64, 32), (6, 4, 1, 256, 16), (17, 2, 2, 72, 4),
                                              (32, 1, 1, 128, 64), (2, 31, 1, 64, 16), (16, 3, 3, 256, 8), (7, 9, 1, 200, 2)])
def test_seventeen_rows_and_more(T, hq, hk, dim, page, lengths, dtype):
    """Two and four row tiles per item at each width, partly empty ones among them."""
    cache, g = _cache(LENGTHS[lengths], T, hk, dim, page, dtype, T * hq + dim, track=True)
    q = torch.randn(cache.batch, T, hq, dim, generator=g, device=DEV).to(dtype)
    out = _check(cache, q)
    _check(cache, q, accumulate=True)
    assert torch.equal(out, cache.attend(q))


def test_token_major_pages_and_scale():
    cache, g = _cache([100, 37], 2, 4, 64, 16, torch.float16, 1, token_major=True)
    _check(cache, torch.randn(2, 2, 8, 64, generator=g, device=DEV).half(), scale=0.05)


def test_pages_the_sequence_does_not_have():
    """Slots of a missing page are not seen; a row that only has such slots is empty."""
    cache, g = _cache([100, 20, 70], 1, 2, 64, 16, torch.float16, 2, track=True)
    cache.block_table[0, 2] = -1
    cache.block_table[0, 4] = cache.num_pages
    cache.block_table[1, :] = -5
    q = torch.randn(3, 1, 4, 64, generator=g, device=DEV).half()
    out = _check(cache, q, accumulate=True)
    assert (out[1] == 0).all()


def test_lengths_past_the_capacity():
    """Lengths are device data: one that passes the table is cut to it."""
    cache, g = _cache([60, 10], 1, 2, 64, 16, torch.float16, 3, garbage=0.5)
    q = torch.randn(2, 1, 4, 64, generator=g, device=DEV).half()
    cache.lengths.copy_(torch.tensor([2 ** 31 - 1, 10], dtype=torch.int32))
    _check(cache, q)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("T,hq,hk", [(4, 8, 2), (4, 16, 1), (8, 64, 8), (5, 20, 1), (20, 4, 4)])
def test_later_drafts_do_not_reach_earlier_rows(T, hq, hk, bad):
    """A drafted token whose key or value is not finite leaves the tokens before it as they are."""
    cache, g = _cache([77], T, hk, 64, 16, torch.float16, 4)
    q = torch.randn(1, T, hq, 64, generator=g, device=DEV).half()
    clean = cache.attend(q)
    at = 77 + T - 2  # the last token but one
    page, off = int(cache.block_table[0, at // 16]), at % 16
    for x in (cache.k_pages, cache.v_pages):
        keep = x[0, page, :, off].clone()
        x[0, page, :, off] = bad
        out = cache.attend(q)
        assert torch.equal(out[:, :T - 2], clean[:, :T - 2])
        x[0, page, :, off] = keep


def test_scores_at_the_type_s_ends():
    """Scores of the lowest and highest values, equal maxima, and very peaked rows."""
    cache, g = _cache([40], 1, 1, 64, 16, torch.float16, 5)
    q = torch.randn(1, 1, 2, 64, generator=g, device=DEV).half()
    page = cache.block_table[0].long()
    cache.k_pages[0, page[0], 0, 3] = q[0, 0, 0] * 60  # one slot takes all the weight
    _check(cache, q, E=2.0 ** -20 * 60 / 8 * float(q[0, 0, 0].double().square().sum()))
    cache.k_pages[0].copy_(torch.full_like(cache.k_pages[0], -65504.0))
    q.fill_(65504.0)
    out, lse = cache.attend(q, return_lse=True)  # every score -3.4e10: equal weights
    mean = torch.stack([R.slots_of(cache.v_pages[0], cache.block_table[0], 41)[0][:, 0].double().mean(0)] * 2)
    assert torch.allclose(out[0, 0].double(), mean, rtol=2e-3, atol=1e-4)
    ref = -64 * 65504.0 ** 2 / 8 + math.log(41)
    assert float((lse.double() - ref).abs().max()) <= abs(ref) * 2.0 ** -22


def test_many_sequences():
    """More sequences than one block of the scan, with idle ones among them."""
    lengths = [(-1 if i % 7 == 3 else (i * 37) % 150) for i in range(300)]
    cache, g = _cache(lengths, 1, 2, 64, 16, torch.float16, 6, track=True)
    _check(cache, torch.randn(300, 1, 8, 64, generator=g, device=DEV).half(), accumulate=True)


def test_workspace_is_fit_for_other_sizes():
    """One cache, calls of different sizes in turn: the shared workspace carries nothing over."""
    cache, g = _cache([900, 20, 1500], 9, 2, 64, 16, torch.float16, 7, track=True)
    q = torch.randn(3, 9, 16, 64, generator=g, device=DEV).half()
    for T, hq, acc in ((1, 4, False), (9, 16, True), (2, 2, False), (9, 8, False), (1, 16, True), (1, 4, False)):
        part = q[:, :T, :hq]
        _check(cache, part, accumulate=acc)


def test_streams_and_graph():
    cache, g = _cache([300, 40], 1, 2, 128, 16, torch.float16, 8)
    q = torch.randn(2, 1, 8, 128, generator=g, device=DEV).half()
    want = cache.attend(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = cache.attend(q)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for n in (300, 10, 200):  # lengths are read on the device, also in a replay
        cache.lengths[0] = n
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, cache.attend(q))
        torch.cuda.synchronize()


def test_lengths_changed_between_calls():
    """Lengths written by the kernel just before the call count in both of its launches."""
    cache, g = _cache([640, 640, 640], 1, 2, 128, 16, torch.float16, 9, track=True)
    q = torch.randn(3, 1, 8, 128, generator=g, device=DEV).half()
    lens = torch.randint(0, 640, (40, 3), generator=g, device=DEV, dtype=torch.int32)
    cache.attend(q, accumulate=True)
    torch.cuda.synchronize()
    sums = []
    for i in range(len(lens)):
        cache.scores.zero_()
        cache.lengths.copy_(lens[i])
        cache.attend(q, accumulate=True)
        sums.append((cache.scores[0].sum(-1), (cache.scores[0] > 0).sum(-1)))
    for i, (weight, count) in enumerate(sums):
        assert float((weight - 4).abs().max()) < 1e-3  # four rows of weight one on each kv head
        assert (count <= lens[i][:, None] + 1).all()


def test_status_word():
    """A wait that gave up is reported once (from a host-written record: the
    status word behind the 512 counters) and the workspace stays fit."""
    cache, g = _cache([50], 1, 2, 64, 16, torch.float16, 10)
    cache.status()  # before any call
    q = torch.randn(1, 1, 4, 64, generator=g, device=DEV).half()
    want = cache.attend(q)
    cache.status()
    cache._ws[2048] = 1
    with pytest.raises(RuntimeError, match="wait"):
        cache.status()
    cache.status()
    assert torch.equal(cache.attend(q), want)


def test_refusals():
    from turbopress_b200 import _abi
    from turbopress_b200.paged import PagedKVCache
    cache = PagedKVCache(2, 2, 64, 4, 16, 2)
    q = torch.zeros(2, 1, 4, 64, device=DEV).half()
    for bad in (lambda: cache.attend(q[:1]), lambda: cache.attend(q[..., :32]), lambda: cache.attend(q.float()),
                lambda: cache.attend(q[:, :, :3]), lambda: cache.attend(q.cpu()), lambda: cache.attend(q, accumulate=True),
                lambda: cache.attend(q, layer=-1), lambda: cache.attend(q[0])):
        with pytest.raises(ValueError):
            bad()
    assert cache.attend(q[:, :0]).shape == (2, 0, 4, 64)
    pages = torch.zeros(4, 2, 16, 64, device=DEV).half()
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in ((pages.float(), pages.float(), table, lens), (pages, pages[:2], table, lens), (pages, pages, table.long(), lens),
                (pages, pages, table, lens.long()), (pages, pages, table, lens[:1]),
                (pages[..., ::2], pages[..., ::2], table, lens)):
        with pytest.raises(ValueError):
            PagedKVCache.from_tensors(*bad)
    with pytest.raises(RuntimeError):
        PagedKVCache.from_tensors(pages.cpu(), pages.cpu(), table.cpu(), lens.cpu())
    odd = torch.zeros(4, 2, 12, 64, device=DEV).half()
    with pytest.raises(RuntimeError):  # page sizes are powers of two
        PagedKVCache.from_tensors(odd, odd, table, lens).attend(q)
    shifted = torch.zeros(4 * 2 * 16 * 64 + 8, device=DEV).half()[4:-4].view(4, 2, 16, 64)
    with pytest.raises(ValueError):  # 8-byte alignment
        PagedKVCache.from_tensors(shifted, shifted, table, lens).attend(q)
    lib = _abi.lib()
    assert lib.tp_paged_attn(None, None, None, 0, None) == _abi.TP_ERR_ARG
    assert lib.tp_paged_attn_workspace_bytes(None, 1, 1, 0) < 0
