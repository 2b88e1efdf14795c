"""GPU tests of the accumulated attention weights (``PagedKVCache.attend`` with
``accumulate``) over prompt chunks: values against a 64-bit restatement, and the
workspace.

Tolerance: as ``tests/test_gpu_paged_attn.py`` has it: E = 1e-5 in a score, so a
slot's weight within 4 E of its value; its sum in 32 bits (at most 32 terms in one
chain, then the chains: 2^-24 * (32 + rows / 512 + 3) < 1e-5 below 40000 rows); and
the rounding of the total.
"""

import ctypes

import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 1e-5


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _cache(lengths, T, hk, dim, page, dtype, seed, spare=3):
    """Random keys and values in every slot, pages in random order, `spare` pages' worth of capacity past the longest."""
    from turbopress_b200.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(seed)
    counts = [max(1, -(-(max(0, n) + T) // page)) for n in lengths]
    P, maxp = sum(counts) + 1, max(counts) + spare
    kp, vp = (torch.randn(P, hk, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    order = torch.randperm(P, generator=g, device=DEV).int()
    table = torch.full((len(lengths), maxp), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    scores = torch.rand(len(lengths), hk, maxp * page, generator=g, device=DEV) * 0.01
    cache = PagedKVCache.from_tensors(kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scores=scores)
    return cache, g


def _weights(q, cache, counts=None):
    """Each slot's weight over the first `counts` tokens of each sequence, float64."""
    B, T, hq, D = q.shape
    hk, cap, g = cache.kv_heads, cache.capacity, hq // cache.kv_heads
    w = torch.zeros(B, hk, cap, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = int(cache.lengths[b])
        used = T if counts is None else max(0, min(T, int(counts[b])))
        if n < 0 or used == 0:
            continue
        end = min(n + used, cap)
        k, ok = R.slots_of(cache.k_pages[0], cache.block_table[b], end)
        see = (torch.arange(end, device=DEV) < n + 1 + torch.arange(used, device=DEV)[:, None]) & ok
        for h in range(hk):
            s = torch.einsum("tgd,sd->tgs", q[b, :used, h * g:(h + 1) * g].double(), k[:, h].double()) * D ** -0.5
            p = torch.softmax(s.masked_fill(~see[:, None], float("-inf")), -1).nan_to_num(0.0)
            w[b, h, :end] = p.sum((0, 1))
    return w


def _check(cache, before, want):
    got = cache.scores[0].double() - before.double()
    lim = (4 * E + 1e-5) * want + 2.0 ** -23 * cache.scores[0].double().abs() + 1e-30
    assert not (~((got - want).abs() <= lim)).any(), float(((got - want).abs() / lim).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[0], [700, -1, 0, 33, 64], [1500]])
@pytest.mark.parametrize("T,hq,hk,dim,page", [(33, 4, 4, 128, 16), (9, 8, 2, 64, 8), (200, 12, 2, 80, 16), (64, 7, 1, 256, 1),
                                              (129, 32, 8, 128, 64), (17, 2, 1, 8, 4)])
def test_weights_of_a_chunk(T, hq, hk, dim, page, lengths, dtype):
    cache, g = _cache(lengths, T, hk, dim, page, dtype, T + hq)
    cache.block_table[0, 2] = -1  # a page it does not have
    q = torch.randn(len(lengths), T, hq, dim, generator=g, device=DEV).to(dtype)
    before = cache.scores[0].clone()
    plain = cache.attend(q)
    assert torch.equal(before, cache.scores[0])
    out = cache.attend(q, accumulate=True)
    assert torch.equal(out, plain)
    want = _weights(q, cache)
    _check(cache, before, want)
    first = cache.scores[0].clone()
    cache.scores[0].copy_(before)
    cache.attend(q, accumulate=True)
    assert torch.equal(first, cache.scores[0])


def test_a_key_that_is_not_finite_stays_with_its_slot_s_rows():
    """A drafted key of NaN: the rows before it add their weights to the slots
    that they see, and the slots past the sequence keep what they hold."""
    cache, g = _cache([50], 40, 1, 64, 16, torch.float16, 3)
    q = torch.randn(1, 40, 2, 64, generator=g, device=DEV).half()
    for s in range(90, cache.capacity):  # unseen slots hold anything
        page_id = int(cache.block_table[0, s // 16])
        if page_id >= 0:
            cache.k_pages[0, page_id, :, s % 16] = float("nan")
    before = cache.scores[0].clone()
    cache.attend(q, accumulate=True)
    _check(cache, before, _weights(q, cache))
    assert torch.equal(cache.scores[0, :, :, 90:], before[:, :, 90:])


def test_workspace_of_long_chunks():
    """The workspace of a call with weights: the rows' statistics beside the
    call's without, and at most 1 GiB of stored scores for a few rows."""
    from turbopress_b200 import _abi
    from turbopress_b200.paged import PagedKVCache
    cache = PagedKVCache(8, 8, 128, 4, 16, 512)  # 8192 slots per sequence
    lib, addr = _abi.lib(), ctypes.addressof(cache._structs[0])
    for tokens in (1, 8, 9, 512, 2048, 8192):
        with_w, without = (lib.tp_paged_attn_workspace_bytes(addr, tokens, 32, acc) for acc in (1, 0))
        assert 0 < without <= with_w
        rows = tokens * 4
        stored = 8 * 8 * (8192 // 128 + 2) * 128 * (16 if rows <= 16 else 32) * 4 if rows <= 32 else 0
        assert with_w - without <= 8 * tokens * 32 * 4 + stored + 1024
    wide = PagedKVCache(64, 8, 128, 4, 16, 1 << 14)  # 262144 slots: 8.6 GB of scores of 16 rows
    assert lib.tp_paged_attn_workspace_bytes(ctypes.addressof(wide._structs[0]), 1, 32, 1) < 64 << 20


def test_capacity_past_the_stored_scores():
    """One row over a capacity whose stored scores would pass 1 GiB: the same weights from K."""
    cache, g = _cache([300, 5], 1, 1, 64, 64, torch.float16, 5, spare=(1 << 24) // 64)
    q = torch.randn(2, 1, 4, 64, generator=g, device=DEV).half()
    before = cache.scores[0].clone()
    cache.attend(q, accumulate=True)
    assert cache._ws.numel() < 64 << 20
    want = _weights_small(q, cache)
    got = cache.scores[0, :, :, :512].double() - before[:, :, :512].double()
    assert ((got - want).abs() <= (4 * E + 1e-5) * want + 2.0 ** -23 * cache.scores[0, :, :, :512].double().abs()).all()
    assert torch.equal(cache.scores[0, :, :, 512:], before[:, :, 512:])


def _weights_small(q, cache):
    w = torch.zeros(q.shape[0], 1, 512, dtype=torch.float64, device=DEV)
    for b in range(q.shape[0]):
        n = int(cache.lengths[b]) + 1
        k, _ = R.slots_of(cache.k_pages[0], cache.block_table[b], n)
        w[b, 0, :n] = torch.softmax(q[b, 0].double() @ k[:, 0].double().T * q.shape[3] ** -0.5, -1).sum(0)
    return w


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,hq,hk,dim,page", [(1, 8, 2, 64, 16), (5, 16, 8, 128, 32), (40, 4, 1, 256, 8), (300, 3, 3, 72, 16)])
def test_weights_of_the_tokens_that_stand(T, hq, hk, dim, page, dtype):
    """add_weights takes each sequence's first tokens, and with all of them is what accumulate adds."""
    lengths = [150, 0, -1, 64, 7, 1000]
    cache, g = _cache(lengths, T, hk, dim, page, dtype, T + dim)
    q = torch.randn(len(lengths), T, hq, dim, generator=g, device=DEV).to(dtype)
    before = cache.scores[0].clone()
    out, lse = cache.attend(q, return_lse=True)
    for counts in (None, torch.tensor([T, 0, T, 1, max(1, T // 2), T + 9], dtype=torch.int32, device=DEV),
                   torch.tensor([-4, 1, 1, T, T, 0], dtype=torch.int32, device=DEV)):
        cache.scores[0].copy_(before)
        cache.add_weights(q, lse, counts)
        _check(cache, before, _weights(q, cache, counts))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # views are taken as they are, on another stream
        cache.scores[0].copy_(before)
        wide = torch.stack((q, q), -2).flatten(2, 3)[:, :, ::2]
        cache.add_weights(wide, torch.stack((lse, lse), -1)[..., 0], scale=0.03)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.isfinite(cache.scores[0]).all()


def test_add_weights_refusals():
    from turbopress_b200 import _abi
    from turbopress_b200.paged import PagedKVCache
    cache = PagedKVCache(2, 2, 64, 4, 16, 2, track_weights=True)
    q, lse = torch.zeros(2, 3, 4, 64, device=DEV).half(), torch.zeros(2, 3, 4, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: cache.add_weights(q[:1], lse[:1]), lambda: cache.add_weights(q.float(), lse), lambda: cache.add_weights(q, lse[:, :2]),
                lambda: cache.add_weights(q, lse.double()), lambda: cache.add_weights(q, lse, n.long()), lambda: cache.add_weights(q, lse, n[:1]),
                lambda: cache.add_weights(q, lse, n.cpu()), lambda: cache.add_weights(q, lse, layer=1),
                lambda: cache.add_weights(q[:, :, :3], lse[:, :, :3]),
                lambda: PagedKVCache(2, 2, 64, 4, 16, 2).add_weights(q, lse)):
        with pytest.raises(ValueError):
            bad()
    cache.add_weights(q[:, :0], lse[:, :0])
    assert _abi.lib().tp_paged_weights(None, None, None) == _abi.TP_ERR_ARG
    assert (cache.scores == 0).all()


def _decoder(batch, seed=3):
    import numpy as np

    from tests.conftest import GOLDEN
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.paged_decoder import PagedDecoder
    from turbopress_b200.synthetic import step_config, synthetic_decoder
    cfg = dict(name="test", layers=2, hidden=1024, inter=2048, q_heads=16, kv_heads=8, head_dim=128, rope_theta=1_000_000.0,
               qk_norm=True)
    with np.load(GOLDEN / "codebooks.npz") as f:
        cbs = {3: torch.from_numpy(f["opt_b3_s64"])}
    layers, fnorm = synthetic_decoder(cfg, [3, 3], cbs, DEV, seed=seed)
    cache = PagedKVCache(batch, 8, 128, batch * 8, 16, 8, layers=2, track_weights=True)
    cache.block_table.copy_(torch.arange(batch * 8, device=DEV).view(batch, 8))
    return PagedDecoder(layers, step_config(cfg), fnorm, cache)


@pytest.mark.parametrize("ragged", [False, True])
def test_rejected_drafts_leave_no_weights(ragged):
    """A bounded cache's weights after rounds with wrong drafts are those of the
    emitted tokens alone, taken one by one (1 % of a weight: the linears of one
    and of five rows round apart; the drafts' rows would add several times
    that)."""
    from turbopress_b200.speculative import DraftVerifier
    g = torch.Generator(device=DEV).manual_seed(5)
    V, B = 500, 2
    emb = torch.randn(V, 1024, generator=g, device=DEV).half()
    head = (emb * 0.05).contiguous()
    prompt = torch.randint(0, V, (B, 40), generator=g, device=DEV)
    none = torch.zeros(B, 0, dtype=torch.int64, device=DEV)
    alone, drafting = _decoder(B), _decoder(B)
    for dec in (alone, drafting):
        dec.step(torch.nn.functional.embedding(prompt, emb), accumulate=True)
        dec.cache.advance(40)
    last = torch.tensor([3, 4], device=DEV)
    plain, ver = [last.tolist()], DraftVerifier(B, 0, V)
    for _ in range(3):
        _, out = alone.speculative_step(last, none, emb, head, ver, accumulate=True)
        last = out[:, 0].contiguous()
        plain.append(last.tolist())
    # the same three tokens in one round: two drafts that stand and two that do not (or are not in use)
    drafts = torch.tensor([[plain[1][b], plain[2][b], (plain[3][b] + 1) % V, 7] for b in range(B)], device=DEV)
    counts = torch.tensor([2, 4], dtype=torch.int32, device=DEV) if ragged else None
    accepted, out = drafting.speculative_step(torch.tensor(plain[0], device=DEV), drafts, emb, head, DraftVerifier(B, 4, V),
                                              accumulate=True, n_drafts=counts)
    assert accepted.tolist() == [2, 2] and out[:, 2].tolist() == plain[3]
    assert torch.equal(alone.cache.lengths, drafting.cache.lengths)
    a, d = alone.cache.scores, drafting.cache.scores
    assert (a[..., 43:] == 0).all() and (d[..., 43:] == 0).all()
    assert float(((a - d).abs() / a.clamp(min=0.05))[..., :43].max()) < 1e-2
