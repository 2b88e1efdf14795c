"""GPU tests of ``PagedKVCache.attend`` at the ends of what a probability and a
value can be, against a 64-bit restatement."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _shared(n, batch, kv_heads, dim, page, dtype):
    """Zeroed pages of n slots that `batch` sequences share (attention only reads them)."""
    from turbopress_b200.paged import PagedKVCache
    P = -(-n // page)
    kp, vp = (torch.zeros(P, kv_heads, page, dim, dtype=dtype, device=DEV) for _ in range(2))
    table = torch.arange(P, dtype=torch.int32, device=DEV).repeat(batch, 1)
    return PagedKVCache.from_tensors(kp, vp, table, torch.full((batch,), n - 1, dtype=torch.int32, device=DEV)), kp, vp


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nats", [17.5, 21.0])
@pytest.mark.parametrize("heads", [4, 32, 40])
def test_a_flat_tail_below_one_large_score(heads, nats, dtype):
    """One slot (of value 0) takes nearly all the weight, 20000 equal ones share
    the rest: the output is their weight times their mean value.  More
    sequences than the GPU holds blocks, so that one block has all of a row.

    Tolerance, relative to the output, which is a sum of equal signs: half an
    ulp; the scores' error E = 2^-24 * 16 * nats < 2^-15 twice in the
    probability (score and normaliser); 2^-16 for its two terms; the fp32 sum,
    below 20000 / 16 / 2 products in one chain: 2^-24 * 625 < 2^-14.  lse has
    E and the normaliser's chain: one addition per 16 or 32 slots of a warp
    (an eighth of all with 16 rows, half with 64), at most 20000 / 2 / 32 of them.
    """
    n, dim = 20000, 64
    cache, kp, vp = _shared(n, 320, 1, dim, 16, dtype)
    g = torch.Generator(device=DEV).manual_seed(heads)
    vp.copy_((1 + 0.25 * torch.rand(vp.shape, generator=g, device=DEV)).to(dtype))
    kp[0, 0, 0, 0], vp[0, 0, 0] = 8.0, 0.0
    q = torch.zeros(320, 1, heads, dim, dtype=dtype, device=DEV)
    q[..., 0] = nats  # times 8 and the scale 1/8
    out, lse = cache.attend(q, return_lse=True)
    v = vp.transpose(1, 2).reshape(-1, dim)[:n].double()
    top = float(q[0, 0, 0, 0])
    total = 1 + (n - 1) * math.exp(-top)
    want = v[1:].sum(0) * math.exp(-top) / total
    err = (out.double() - want).abs() / want
    assert float(err.max()) <= HALF_ULP[dtype] + 2 * 2.0 ** -15 + 2.0 ** -16 + 2.0 ** -14 + 2.0 ** -25 / float(want.min())
    assert float((lse.double() - (top + math.log(total))).abs().max()) <= 2.0 ** -15


def _values(cache, n):
    from tests import paged_reference as R
    return R.slots_of(cache.v_pages[0], cache.block_table[0], n)[0].double()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,hq,hk,dim,page", [(1, 4, 2, 128, 16), (1, 24, 1, 64, 16), (1, 40, 1, 128, 32), (4, 8, 1, 64, 8), (3, 32, 2, 256, 16),
                                              (5, 20, 2, 72, 4)])
def test_infinite_values_in_seen_slots(T, hq, hk, dim, page, dtype):
    """A value of +-inf gives +-inf to the rows that see its slot (whatever
    the slot's weight: the row's largest, a usual one or a very small one), NaN
    where both signs meet, and nothing to other rows and columns."""
    from tests import paged_reference as R
    from turbopress_b200.paged import PagedKVCache
    g = torch.Generator(device=DEV).manual_seed(T * hq + dim)
    n = 700
    P = -(-(n + T) // page)
    kp, vp = (torch.randn(P, hk, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    table = torch.randperm(P, generator=g, device=DEV).int()[None].contiguous()
    cache = PagedKVCache.from_tensors(kp, vp, table, torch.tensor([n], dtype=torch.int32, device=DEV))
    q = torch.randn(1, T, hq, dim, generator=g, device=DEV).to(dtype)

    def at(slot):  # where a slot lies
        return int(table[0, slot // page]), slot % page

    # one slot with the row's largest score, one 20 nats below the others
    page_id, off = at(40)
    kp[page_id, :, off] = q[0, 0, ::hq // hk][:hk] * 2
    page_id, off = at(41)
    kp[page_id, :, off] = q[0, 0, ::hq // hk][:hk] * -1
    for i, (slot, col, val) in enumerate([(0, 0, math.inf), (40, 1, -math.inf), (41, 2, math.inf), (100, 3, -math.inf), (333, 4, math.inf),
                                          (n - 1, 5, math.inf), (n, 6, -math.inf), (n + T - 1, 7, math.inf), (255, 3, math.inf)]):
        page_id, off = at(slot)
        vp[page_id, :, off, col] = val
    out = cache.attend(q)
    want, _, _ = R.attention(q, kp, vp, table, cache.lengths)
    assert torch.isinf(want).any() and torch.isnan(want[..., 3]).all()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    sign = torch.where(torch.isinf(want), want.sign(), 0.0)
    assert torch.equal(torch.where(torch.isinf(out), out.sign(), 0.0).double(), sign)
    fine = torch.isfinite(want)
    tol = HALF_ULP[dtype] * want.abs() * (1 + 2.0 ** -6) + 4 * 2.0 ** -15 * 6
    assert ((out.double() - want).abs() <= tol)[fine].all()
