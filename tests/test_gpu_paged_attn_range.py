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
