"""GPU tests of ``tp_verify_drafts`` (``DraftVerifier``) against a 64-bit
restatement.

The outputs are whole numbers and must be equal.  Probabilities are good to
about 2^-20 relative in 32 bits, so a comparison nearer to equality than 1e-5
could go either way: such inputs are skipped by the restatement's own margin
(and at most one in twenty may be).
"""

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


def _inputs(B, K, V, dtype, seed, probs, heat, ragged=False, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    target = torch.randn(B, K + 1, V, generator=g, device=DEV) * spread
    draft = target[:, :K] + 0.7 * torch.randn(B, K, V, generator=g, device=DEV)
    x = dict(logits=target.to(dtype), uniforms=torch.rand(B, K, generator=g, device=DEV),
             noise=torch.empty(B, V, device=DEV).exponential_(generator=g), draft_probs=None, n_drafts=None,
             temperature=torch.full((B,), heat, device=DEV))
    q = torch.softmax(draft / (heat or 1.0), -1)
    if probs:
        x["draft_probs"] = q.contiguous()
        x["draft_tokens"] = (q / torch.empty_like(q).exponential_(generator=g)).argmax(-1)
    else:
        x["draft_tokens"] = draft.argmax(-1)
    if ragged:
        x["n_drafts"] = torch.randint(0, K + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    return x


def _check(x, verifier=None):
    from turbopress_b200.speculative import DraftVerifier
    B, rows, V = x["logits"].shape
    verifier = verifier or DraftVerifier(B, rows - 1, V)
    ref = R.verify(x["logits"], x["draft_tokens"], x["uniforms"], x["noise"], x["draft_probs"], x["temperature"], x["n_drafts"])
    for _ in range(2):  # the workspace is left fit
        accepted, tokens = verifier(**x)
        if ref[2] > 1e-5:
            assert accepted.tolist() == ref[0].tolist()
            assert tokens.tolist() == ref[1].tolist()
    return ref


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V", [(1, 4, 151936), (5, 3, 5003), (3, 8, 1000), (40, 1, 257), (2, 63, 130), (1, 0, 9), (4, 2, 1),
                                   (2, 5, 7), (70, 2, 2049)])
def test_verify(B, K, V, dtype):
    skipped = 0
    for seed, (probs, heat, ragged) in enumerate([(True, 1.0, False), (False, 0.7, False), (True, 0.8, True), (False, 0.0, True)]):
        skipped += _check(_inputs(B, K, V, dtype, seed + B + K + V, probs, heat, ragged))[2] <= 1e-5
    assert skipped <= 1


def test_mixed_temperatures():
    for seed in range(4):
        x = _inputs(9, 4, 4001, torch.float16, 50 + seed, True, 1.0)
        x["temperature"] = torch.tensor([0, 1, 0.5, 0, 2, 0.1, 100, 0, 1e-3], device=DEV)
        _check(x)


def test_low_temperatures_keep_their_digits():
    """Acceptance at the edge: at temperature 1e-3 two near logits share the
    probability; uniforms 1e-3 relative below and above p decide (fp32 logits
    near 20 make m / t about 2^15, so p depends on x - m being taken first)."""
    from turbopress_b200.speculative import DraftVerifier
    x = _inputs(2, 1, 4096, torch.float32, 60, False, 1e-3)
    g = torch.Generator(device=DEV).manual_seed(60)
    x["logits"] = torch.randn(2, 2, 4096, generator=g, device=DEV)
    x["logits"][:, 0, 100], x["logits"][:, 0, 3000] = 20.0, 20.0 - 4.0e-4
    x["draft_tokens"].fill_(100)
    p = torch.softmax(x["logits"][:, 0].double() / 1e-3, -1)[:, 100]
    x["uniforms"] = torch.stack((p[:1] * (1 - 1e-4), p[1:] * (1 + 1e-4))).float()
    accepted, _ = DraftVerifier(2, 1, 4096)(**x)
    assert accepted.tolist() == [1, 0]


def test_all_greedy_without_random_numbers():
    x = _inputs(3, 4, 5003, torch.bfloat16, 1, False, 0.0)
    x["draft_tokens"][0] = x["logits"][0, :4].float().argmax(-1)
    ref = _check(x)
    x.update(uniforms=None, noise=None, temperature=None)
    from turbopress_b200.speculative import DraftVerifier
    accepted, tokens = DraftVerifier(3, 4, 5003)(**x)
    assert tokens.tolist() == ref[1].tolist() and accepted.tolist() == ref[0].tolist()


def test_greedy_ties_and_values_at_the_ends():
    """Equal maxima take the lower index, a NaN is the maximum, -0 equals 0, all -inf gives token 0."""
    x = _inputs(6, 1, 999, torch.float16, 2, False, 0.0)
    x["logits"].clamp_(-3, 3)
    x["logits"][0, 0, [700, 3, 998]] = 9.0
    x["draft_tokens"][0] = 3
    x["logits"][1, 0, 800] = math.nan
    x["logits"][1, 0, 400] = math.nan
    x["draft_tokens"][1] = 400
    x["logits"][2].fill_(-math.inf)
    x["draft_tokens"][2] = 0
    x["logits"][3].fill_(-1.0)
    x["logits"][3, 0, 5] = -0.0
    x["logits"][3, 0, 2] = -0.0
    x["logits"][3, 0, 9] = 0.0
    x["draft_tokens"][3] = 2
    x["logits"][4, 0, 77] = math.inf
    x["draft_tokens"][4] = 77
    ref = _check(x)
    assert ref[0].tolist()[:5] == [1, 1, 1, 1, 1]


def test_masked_logits():
    """-inf logits (a filtered vocabulary) carry no probability; a draft among them is rejected."""
    x = _inputs(4, 3, 3001, torch.float32, 3, True, 0.9)
    x["logits"][:, :, 50:] = -math.inf
    x["draft_tokens"][0, 0] = 60
    x["draft_tokens"][1] = torch.randint(0, 50, (3,), device=DEV)
    ref = _check(x)
    assert ref[0][0] == 0 and int(ref[1].max()) < 60
    one = _inputs(1, 2, 500, torch.float16, 4, False, 1.0)
    one["logits"].fill_(-math.inf)
    one["logits"][..., 123] = 1.0
    one["draft_tokens"].fill_(123)
    assert _check(one)[1].tolist() == [[123, 123, 123]]


def test_rows_without_probability():
    from turbopress_b200.speculative import DraftVerifier
    x = _inputs(2, 2, 500, torch.float32, 5, False, 1.0)
    x["logits"].fill_(-math.inf)
    x["logits"][1].fill_(math.nan)
    accepted, tokens = DraftVerifier(2, 2, 500)(**x)
    assert accepted.tolist() == [0, 0] and tokens.tolist() == [[-1] * 3] * 2


def test_drafts_outside_the_vocabulary():
    x = _inputs(3, 3, 700, torch.float32, 6, False, 1.0)
    x["draft_tokens"][0, 0] = -1
    x["draft_tokens"][1, 1] = 700
    x["draft_tokens"][2, 2] = 1 << 40
    _check(x)
    x["draft_probs"] = torch.softmax(torch.randn(3, 3, 700, device=DEV), -1)
    _check(x)
    x["temperature"].zero_()
    _check(x)


def test_equal_distributions():
    """q = p: every draft stands; q >= p everywhere (a q that is not normalised): drawn from p."""
    x = _inputs(2, 3, 400, torch.float32, 7, True, 1.0)
    x["draft_probs"] = (torch.softmax(x["logits"][:, :3].double(), -1)).float().contiguous()
    x["uniforms"].clamp_(max=0.99)
    assert _check(x)[0].tolist() == [3, 3]
    x["draft_probs"].mul_(2.0)
    x["uniforms"].fill_(0.75)  # 0.75 * 2 p >= p: rejected, nothing left of p - 2 p
    ref = _check(x)
    assert ref[0].tolist() == [0, 0] and int(ref[1][:, 0].min()) >= 0


def test_uniform_zero_and_noise_at_the_ends():
    x = _inputs(3, 2, 600, torch.float32, 8, True, 1.0)
    x["uniforms"].zero_()  # 0 < p: accepted
    assert _check(x)[0].tolist() == [2, 2, 2]
    x["uniforms"].fill_(1.0 - 2.0 ** -24)
    x["noise"][0, 17] = 0.0  # wins the race where it has any probability
    x["noise"][1].fill_(3e38)
    x["noise"][1, 44] = 1e-30
    _check(x)


def test_strided_logits():
    """Padded vocabularies and rows whose addresses are aligned to one element only."""
    for dtype, pad in ((torch.float16, 5), (torch.bfloat16, 1), (torch.float32, 3)):
        x = _inputs(3, 2, 1001, dtype, 9, True, 1.0)
        wide = torch.full((3, 3, 1001 + pad), math.inf, dtype=dtype, device=DEV)
        wide[..., :1001] = x["logits"]
        x["logits"] = wide[..., :1001]
        _check(x)
        wide = torch.full((3, 3, 1001 + pad), math.nan, dtype=dtype, device=DEV)
        wide[..., pad:] = x["logits"]
        x["logits"] = wide[..., pad:]
        _check(x)


def test_one_verifier_for_smaller_calls():
    from turbopress_b200.speculative import DraftVerifier
    verifier = DraftVerifier(8, 5, 3000)
    for seed, (B, K) in enumerate([(8, 5), (1, 1), (3, 5), (8, 0), (2, 3), (8, 5)]):
        _check(_inputs(B, K, 3000, torch.float16, 20 + seed, True, 1.0, ragged=seed % 2 == 1), verifier)


def test_tokens_follow_the_target():
    """Speculative tokens are distributed as the target's: frequencies of the
    first token over many runs against softmax (5 standard deviations)."""
    from turbopress_b200.speculative import DraftVerifier
    n, V = 20000, 11
    g = torch.Generator(device=DEV).manual_seed(30)
    p_logit, q_logit = torch.randn(V, generator=g, device=DEV), torch.randn(V, generator=g, device=DEV)
    q = torch.softmax(q_logit, -1)
    drafts = (q / torch.empty(n, 1, V, device=DEV).exponential_(generator=g)).argmax(-1)
    logits = torch.stack((p_logit, torch.zeros_like(p_logit))).expand(n, 2, V).contiguous()
    verifier = DraftVerifier(n, 1, V)
    p = torch.softmax(p_logit.double(), -1)
    for probs in (q.expand(n, 1, V).contiguous(), None):
        _, tokens = verifier(logits, drafts, uniforms=torch.rand(n, 1, generator=g, device=DEV),
                             noise=torch.empty(n, V, device=DEV).exponential_(generator=g), draft_probs=probs,
                             temperature=torch.ones(n, device=DEV))
        if probs is None:  # the draft was fixed by its position: compare with what a one-hot q gives
            same = drafts[:, 0] == tokens[:, 0]
            assert abs(float(same.double().mean()) - float(p[drafts[:, 0]].mean())) < 5 * 0.5 / math.sqrt(n)
            continue
        freq = torch.bincount(tokens[:, 0], minlength=V).double() / n
        assert (((freq - p) / (p * (1 - p) / n).sqrt()).abs() < 5).all()


def test_graph():
    x = _inputs(4, 3, 5003, torch.float16, 40, True, 1.0)
    from turbopress_b200.speculative import DraftVerifier
    verifier = DraftVerifier(4, 3, 5003)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        accepted, tokens = verifier(**x)
    for seed in (41, 42):
        y = _inputs(4, 3, 5003, torch.float16, seed, True, 1.0)
        for k, t in x.items():
            if t is not None:
                t.copy_(y[k])
        graph.replay()
        torch.cuda.synchronize()
        ref = R.verify(*(x[k] for k in ("logits", "draft_tokens", "uniforms", "noise", "draft_probs", "temperature", "n_drafts")))
        assert ref[2] <= 1e-5 or (tokens.tolist() == ref[1].tolist() and accepted.tolist() == ref[0].tolist())


def test_refusals():
    from turbopress_b200 import _abi
    from turbopress_b200.speculative import DraftVerifier
    x = _inputs(2, 3, 100, torch.float16, 10, True, 1.0)
    verifier = DraftVerifier(2, 3, 100)
    for key, val in (("logits", x["logits"][..., :99]), ("logits", x["logits"][0]), ("logits", x["logits"].double()),
                     ("logits", x["logits"].cpu()), ("draft_tokens", x["draft_tokens"].int()),
                     ("draft_tokens", x["draft_tokens"][:, :2]), ("uniforms", None), ("noise", None),
                     ("noise", x["noise"][:, ::2]), ("draft_probs", x["draft_probs"].half()),
                     ("temperature", torch.ones(3, device=DEV)), ("n_drafts", torch.zeros(2, dtype=torch.int64, device=DEV)),
                     ("logits", x["logits"].transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            verifier(**{**x, key: val})
    with pytest.raises(ValueError):
        verifier(**_inputs(3, 3, 100, torch.float16, 10, True, 1.0))
    with pytest.raises(RuntimeError):
        DraftVerifier(1, 64, 100)
    with pytest.raises(ValueError):
        DraftVerifier(0, 1, 100)
    assert _abi.lib().tp_verify_drafts(None, None, 0, None) == _abi.TP_ERR_ARG
