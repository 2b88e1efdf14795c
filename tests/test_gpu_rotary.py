"""GPU tests of ``tp_rotary`` (``Rotary`` and ``PagedKVCache.append``) against
a 64-bit restatement.

Tolerances: one rounding to the output type (half an ulp, 2^-11 / 2^-8 / 2^-24
relative for fp16 / bf16 / fp32) and the fp32 arithmetic before it.  A turned
element is a sum of two products of values up to A = |x_i| + |x_j| (times the
scale and the norm's factor) with cos and sin good to 2^-22 (sincospif of an
fp32 angle), so its error before rounding is below 2^-20 A; fp16 adds 2^-25
where the result is subnormal.
"""

import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _near(got, ref, dtype):
    size = ref.abs().amax(-1, keepdim=True)  # bounds every A of the head up to a factor 4
    tol = HALF_ULP[dtype] * ref.abs() * (1 + 2.0 ** -6) + 2.0 ** -18 * size + 2.0 ** -25
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))


def _inputs(shape_q, shape_k, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape_q, generator=g, device=DEV).to(dtype), torch.randn(shape_k, generator=g, device=DEV).to(dtype),
            g)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot,interleaved", [
    (1, 32, 8, 128, 128, False), (1, 32, 8, 128, 128, True), (7, 16, 8, 128, 64, False), (1000, 5, 1, 64, 64, True),
    (333, 12, 4, 96, 96, False), (37, 7, 1, 80, 40, False), (37, 7, 1, 80, 40, True), (2, 4, 4, 256, 256, False),
    (65, 3, 3, 250, 90, True), (65, 3, 3, 250, 90, False), (9, 1, 1, 2, 2, False), (5, 2, 2, 256, 2, True)])
def test_rotary(tokens, hq, hk, dim, rot, interleaved, dtype):
    from turbopress_b200.rotary import Rotary, rope_frequencies
    q, k, g = _inputs((tokens, hq, dim), (tokens, hk, dim), dtype, tokens + dim)
    inv, _ = rope_frequencies(rot, 500000.0)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device=DEV)
    rotary = Rotary(dim, inv, interleaved=interleaved, scale=1.25)
    yq, yk = rotary(q, k, pos)
    assert yq.dtype == dtype and yq.shape == q.shape and yk.shape == k.shape
    _near(yq, R.rotate(q, pos, inv, 1.25, interleaved), dtype)
    _near(yk, R.rotate(k, pos, inv, 1.25, interleaved), dtype)


@pytest.mark.parametrize("dim,rot,interleaved", [(128, 128, False), (128, 32, True), (80, 40, False), (250, 90, True)])
@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_head_norm(dim, rot, interleaved, which):
    from turbopress_b200.rotary import Rotary
    q, k, g = _inputs((3, 5, 6, dim), (3, 5, 2, dim), torch.float16, dim)
    q, k = q * 3, k * 0.01
    wq = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).half() if which != "k" else None
    wk = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).half() if which != "q" else None
    pos = torch.randint(0, 5000, (3, 5), generator=g, device=DEV)
    rotary = Rotary(dim, theta=10000.0, rot_dim=rot, interleaved=interleaved)
    yq, yk = rotary(q, k, pos, q_norm=wq, k_norm=wk, eps=1e-5)
    _near(yq, R.rotate(q, pos, rotary.inv_freq, 1.0, interleaved, weight=wq, eps=1e-5), torch.float16)
    _near(yk, R.rotate(k, pos, rotary.inv_freq, 1.0, interleaved, weight=wk, eps=1e-5), torch.float16)


def test_angles_of_long_contexts():
    """Positions up to 2^31 and below zero: the angle keeps its fraction of a turn."""
    from turbopress_b200.rotary import Rotary
    inv = torch.tensor([1.0, 0.3, 1e-3, 1e-6])
    pos = torch.tensor([0, 1, -1, 131071, 10_000_019, (1 << 31) - 1, -(1 << 31), (1 << 40) + 3], device=DEV)
    x = torch.ones(pos.numel(), 1, 8, device=DEV)
    y, _ = Rotary(8, inv)(x, x, pos)
    _near(y, R.rotate(x, pos, inv), torch.float32)


def test_inverse_is_the_gradient():
    """d<w, rot(x)>/dx = rot^-1(w), also against differences of the 64-bit form."""
    from turbopress_b200.rotary import Rotary
    x, w, g = _inputs((4, 2, 64), (4, 2, 64), torch.float32, 1)
    pos = torch.randint(0, 3000, (4,), generator=g, device=DEV)
    rotary = Rotary(64, theta=10000.0, rot_dim=32, scale=0.9)
    grad, _ = rotary(w, w, pos, inverse=True)
    back, _ = rotary(rotary(x, x, pos)[0], x, pos, inverse=True)
    unit = torch.ones_like(x)
    unit[..., :32] = 0.81  # scale twice on the turned part
    assert torch.allclose(back, x * unit, rtol=0, atol=2e-6 * float(x.abs().max()))
    step = 1e-3
    for at in ((0, 0, 0), (1, 1, 17), (3, 0, 31), (2, 1, 60)):
        d = torch.zeros_like(x)
        d[at] = step
        hi = (R.rotate(x.double() + d, pos, rotary.inv_freq, 0.9) * w.double()).sum()
        lo = (R.rotate(x.double() - d, pos, rotary.inv_freq, 0.9) * w.double()).sum()
        assert abs(float(hi - lo) / (2 * step) - float(grad[at])) < 1e-5


def test_strides_and_in_place_views():
    """Views of one fused projection, token-strided queries, and unaligned ones."""
    from turbopress_b200.rotary import Rotary
    g = torch.Generator(device=DEV).manual_seed(2)
    fused = torch.randn(6, 9, (4 + 2 + 2) * 64 + 8, generator=g, device=DEV).half()
    q, k = fused[..., 8:8 + 256].unflatten(-1, (4, 64)), fused[..., 264:264 + 128].unflatten(-1, (2, 64))
    pos = torch.randint(0, 999, (6, 9), generator=g, device=DEV)
    rotary = Rotary(64)
    yq, yk = rotary(q, k, pos)
    _near(yq, R.rotate(q, pos, rotary.inv_freq), torch.float16)
    _near(yk, R.rotate(k, pos, rotary.inv_freq), torch.float16)
    odd = fused[..., 3:3 + 256].unflatten(-1, (4, 64))  # 2-byte alignment
    yq, _ = rotary(odd, k, pos)
    _near(yq, R.rotate(odd, pos, rotary.inv_freq), torch.float16)
    spread = torch.randn(6, 9, 4, 128, generator=g, device=DEV).half()[..., ::2]
    yq, _ = rotary(spread, k, pos)
    _near(yq, R.rotate(spread, pos, rotary.inv_freq), torch.float16)


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("dtype,dim,page,norm", [(torch.float16, 128, 16, True), (torch.bfloat16, 64, 1, False),
                                                 (torch.float16, 80, 4, False), (torch.bfloat16, 256, 64, True)])
def test_append(dtype, dim, page, norm, token_major):
    """Keys and values land in their slots; idle sequences, tokens past the
    capacity and pages the sequence does not have are left alone."""
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.rotary import Rotary
    B, T, hq, hk, P, maxp = 5, 6, 6, 2, 40, max(2, 24 // page)
    q, k, g = _inputs((B, T, hq, dim), (B, T, hk, dim), dtype, dim + page)
    v = torch.randn(B, T, hk, dim, generator=g, device=DEV).to(dtype)
    shape = (P, page, hk, dim) if token_major else (P, hk, page, dim)
    kp, vp = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
    if token_major:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    if B * maxp <= P:
        table = torch.randperm(P, generator=g, device=DEV)[:B * maxp].reshape(B, maxp).int()
    else:  # more table entries than pages: only the first ones of each sequence
        table = torch.full((B, maxp), -1, dtype=torch.int32, device=DEV)
        table[:, :8] = torch.randperm(P, generator=g, device=DEV)[:40].reshape(B, 8).int()
    table[3, 0] = P + 5  # not a page of the pool
    cap = maxp * page
    lengths = torch.tensor([0, min(3, cap - 1), -1, 0, cap - 2], dtype=torch.int32, device=DEV)
    scores = torch.rand(B, hk, cap, generator=g, device=DEV)
    places = torch.full((B, hk, cap), -7, dtype=torch.int32, device=DEV)
    nxt = torch.tensor([0, 100, 5, 7, 9], dtype=torch.int32, device=DEV)
    cache = PagedKVCache.from_tensors(kp, vp, table, lengths, scores=scores, positions=places, next_pos=nxt)
    wq, wk = ((1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2))
    rotary = Rotary(dim)
    before = [t.clone() for t in (kp, vp, scores, places)]
    out = cache.append(rotary, q, k, v, q_norm=wq, k_norm=wk)
    pos = nxt.long()[:, None] + torch.arange(T, device=DEV)
    _near(out, R.rotate(q, pos, rotary.inv_freq, weight=wq), dtype)
    rk = R.rotate(k, pos, rotary.inv_freq, weight=wk)
    touched = torch.zeros(P, page, dtype=torch.bool, device=DEV)
    slots = torch.zeros(B, cap, dtype=torch.bool, device=DEV)
    for b in range(B):
        for i in range(T):
            s = int(lengths[b]) + i
            if int(lengths[b]) < 0 or s >= cap:
                continue
            slots[b, s] = True
            assert (places[b, :, s] == int(nxt[b]) + i).all() and (scores[b, :, s] == 0).all()
            page_id = int(table[b, s // page])
            if not 0 <= page_id < P:
                continue
            touched[page_id, s % page] = True
            _near(kp[page_id, :, s % page], rk[b, i], dtype)
            assert torch.equal(vp[page_id, :, s % page], v[b, i])
    rest = ~touched[:, None, :, None]
    assert torch.equal(kp.masked_select(rest), before[0].masked_select(rest))
    assert torch.equal(vp.masked_select(rest), before[1].masked_select(rest))
    keep = ~slots[:, None, :]
    assert torch.equal(scores.masked_select(keep), before[2].masked_select(keep))
    assert torch.equal(places.masked_select(keep), before[3].masked_select(keep))
    # positions given explicitly, on another stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out2 = cache.append(rotary, q, k, v, positions=pos + 11, q_norm=wq, k_norm=wk)
    torch.cuda.current_stream().wait_stream(side)
    _near(out2, R.rotate(q, pos + 11, rotary.inv_freq, weight=wq), dtype)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: the last page is where it should be."""
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.rotary import Rotary
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    P, page, hk, dim = (1 << 32) // (64 * 8 * 128) + 3, 64, 8, 128
    kp = torch.empty(P, hk, page, dim, dtype=torch.float16, device=DEV)
    vp = torch.empty_like(kp)
    table = torch.tensor([[P - 1, P - 2]], dtype=torch.int32, device=DEV)
    cache = PagedKVCache.from_tensors(kp, vp, table, torch.tensor([63], dtype=torch.int32, device=DEV))
    q, k, g = _inputs((1, 2, 8, dim), (1, 2, hk, dim), torch.float16, 3)
    rotary = Rotary(dim)
    kp[-2:].zero_()
    vp[-2:].zero_()
    cache.append(rotary, q, k, k)
    ref = R.rotate(k, torch.tensor([[63, 64]], device=DEV), rotary.inv_freq)
    _near(kp[P - 1, :, 63], ref[0, 0], torch.float16)
    _near(kp[P - 2, :, 0], ref[0, 1], torch.float16)
    assert torch.equal(vp[P - 1, :, 63], k[0, 0]) and torch.equal(vp[P - 2, :, 0], k[0, 1])
    # and read back: two slots seen by token 0 would need 64 filled ones; idle slots stay out through lengths
    cache.lengths.fill_(63)
    kp[P - 1].zero_()
    vp[P - 1].zero_()
    vp[P - 1, :, 63] = k[0, 0]
    kp[P - 2, :, 0], vp[P - 2, :, 0] = 0, k[0, 1]
    out = cache.attend(torch.zeros_like(q))  # equal weights over 64 and 65 slots
    assert torch.allclose(out[0, 0], k[0, 0] / 64, rtol=0, atol=1e-4)
    assert torch.allclose(out[0, 1], (k[0, 0] + k[0, 1]) / 65, rtol=0, atol=2e-4)


def test_calls_of_other_kinds_in_turn():
    """One Rotary and one cache over dtypes, strides and position types in
    turn: what was checked for one call is not taken for another."""
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.rotary import Rotary
    rotary = Rotary(64)
    g = torch.Generator(device=DEV).manual_seed(5)
    base = torch.randn(2, 3, 4, 128, generator=g, device=DEV)
    pos = torch.randint(0, 500, (2, 3), generator=g, device=DEV)
    wide = torch.zeros(2, 6, dtype=torch.int64, device=DEV)
    wide[:, ::2] = pos
    for _ in range(2):
        for dtype in (torch.float16, torch.bfloat16, torch.float32):
            x = base.to(dtype)
            for q, k in ((x[..., :64], x[:, :, :2, 64:]), (x[..., :64].contiguous(), x[:, :, :2, 64:].contiguous()),
                         (x.transpose(0, 1)[..., :64].transpose(0, 1), x[:, :, 1:3, :64]), (x[..., ::2], x[:, :, ::2, 1::2])):
                for p in (pos, pos.int(), wide[:, ::2]):
                    yq, yk = rotary(q, k, p)
                    _near(yq, R.rotate(q, pos, rotary.inv_freq), dtype)
                    _near(yk, R.rotate(k, pos, rotary.inv_freq), dtype)
        with pytest.raises(ValueError):
            rotary(base[..., :64], base[..., 64:], pos.cpu())
        with pytest.raises(ValueError):
            rotary(base[..., :64], base[..., 64:].cpu(), pos)
    cache = PagedKVCache(2, 2, 64, 8, 16, 2)
    cache.block_table.copy_(torch.arange(4, device=DEV).view(2, 2))
    for T in (1, 3, 2, 3):
        q, kv = base[:, :T, :, :64].half(), base[:, :T, :2, 64:].half()
        out = cache.append(rotary, q, kv, kv)
        at = cache.next_pos.long()[:, None] + torch.arange(T, device=DEV)
        _near(out, R.rotate(q, at, rotary.inv_freq), torch.float16)
        cache.advance(T)
    assert cache.lengths.tolist() == [9, 9] == cache.next_pos.tolist()
    with pytest.raises(ValueError):
        cache.append(rotary, base[:, :1, :, :64].bfloat16(), base[:, :1, :2, 64:].bfloat16(), base[:, :1, :2, 64:].bfloat16())
    with pytest.raises(ValueError):
        cache.append(rotary, base[:, :1, :, :64].half(), base[:, :1, :2, 64:].half(), base[:, :1, :2, 64:].half().cpu())


def test_refusals():
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.rotary import Rotary
    rotary = Rotary(64)
    q, k = torch.zeros(2, 3, 4, 64, device=DEV).half(), torch.zeros(2, 3, 2, 64, device=DEV).half()
    pos = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    for bad in (lambda: rotary(q[..., :32], k, pos), lambda: rotary(q, k[:, :2], pos), lambda: rotary(q, k.float(), pos),
                lambda: rotary(q, k, pos[:, :2]), lambda: rotary(q, k, None), lambda: rotary(q.cpu(), k.cpu(), pos.cpu()),
                lambda: rotary(q, k, pos, q_norm=torch.ones(32, device=DEV).half()),
                lambda: rotary(q.to(torch.float64), k.to(torch.float64), pos),
                lambda: Rotary(300), lambda: Rotary(64, rot_dim=66), lambda: Rotary(63), lambda: Rotary(64, torch.ones(2, 2)),
                lambda: Rotary(64, torch.tensor([float("inf")])), lambda: Rotary(64, scaling=dict(rope_type="other"))):
        with pytest.raises(ValueError):
            bad()
    assert rotary(q[:0], k[:0], pos[:0])[0].shape == (0, 3, 4, 64)
    cache = PagedKVCache(2, 2, 64, 4, 16, 2)
    for bad in (lambda: cache.append(rotary, q[:1], k[:1], k[:1]), lambda: cache.append(rotary, q.float(), k.float(), k.float()),
                lambda: cache.append(rotary, q, k, k[:, :2]), lambda: cache.append(rotary, q, k[:, :, :1], k[:, :, :1]),
                lambda: cache.append(rotary, q, k, k, layer=1), lambda: cache.append(Rotary(32), q, k, k)):
        with pytest.raises(ValueError):
            bad()
    assert cache.append(rotary, q[:, :0], k[:, :0], k[:, :0]).shape == (2, 0, 4, 64)
