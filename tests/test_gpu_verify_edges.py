"""GPU tests of ``DraftVerifier`` against a 64-bit restatement, sequence by
sequence: each is compared unless its own nearest comparison is closer to
equality than 1e-5 (probabilities are good to 2^-20 in 32 bits), and of all
sequences one in fifty may be."""

import pytest
import torch

from tests import paged_reference as R
from tests.test_gpu_verify import _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _compare(x, verifier=None):
    """(sequences compared, sequences)."""
    from turbopress_b200.speculative import DraftVerifier
    B, rows, V = x["logits"].shape
    accepted, tokens = (verifier or DraftVerifier(B, rows - 1, V))(**x)
    done = 0
    for b in range(B):
        one = {k: None if t is None else t[b:b + 1] for k, t in x.items()}
        ref = R.verify(*(one[k] for k in ("logits", "draft_tokens", "uniforms", "noise", "draft_probs", "temperature", "n_drafts")))
        if ref[2] > 1e-5:
            done += 1
            assert accepted[b].item() == ref[0].item(), b
            assert tokens[b].tolist() == ref[1][0].tolist(), b
    return done, B


@pytest.mark.parametrize("least", [1e-45, 1e-40, 1e-39, 1.1754944e-38, 1e-37, 1e-30])
def test_the_smallest_temperatures(least):
    """Subnormal temperatures (whose inverse passes fp32's range) and the
    smallest normal ones pick the largest logit, as their limit does."""
    x = _inputs(6, 3, 3001, torch.float32, 11, True, 1.0)
    x["temperature"].fill_(least)
    x["logits"][:, 0].scatter_(1, x["draft_tokens"][:, :1], 50.0)  # a first draft that stands
    done, n = _compare(x)
    assert done == n


def test_every_sequence_of_many_calls():
    """All dtypes, vocabularies and kinds of drafts, one sequence at a time, and how many were compared."""
    done = total = 0
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for B, K, V in ((5, 3, 5003), (3, 8, 1000), (40, 1, 257), (2, 63, 130), (1, 0, 9), (4, 2, 1), (2, 5, 7), (70, 2, 2049), (9, 4, 4001),
                        (3, 4, 40003)):
            for seed, (probs, heat, ragged) in enumerate([(True, 1.0, False), (False, 0.7, False), (True, 0.8, True), (False, 0.0, True)]):
                x = _inputs(B, K, V, dtype, 900 + seed + B + K + V, probs, heat, ragged)
                if B == 9:
                    x["temperature"] = torch.tensor([0, 1, 0.5, 0, 2, 0.1, 100, 0, 1e-3], device=DEV)
                d, n = _compare(x)
                done, total = done + d, total + n
    assert done >= 0.98 * total, (done, total)
