"""GPU tests of ``PagedDecoder.speculative_step`` over token ids that are not in
the vocabulary: padded drafts, and the -1 of a row without probability."""

import importlib.util
from pathlib import Path

import pytest
import torch

from tests.test_gpu_paged_weights import _decoder

pytestmark = pytest.mark.gpu
DEV = "cuda"
V = 500


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def test_ids_outside_the_vocabulary():
    from turbopress_b200.speculative import DraftVerifier
    g = torch.Generator(device=DEV).manual_seed(2)
    emb = torch.randn(V, 1024, generator=g, device=DEV).half()
    head = (emb * 0.05).contiguous()
    plain, padded = _decoder(3), _decoder(3)
    last = torch.tensor([3, 4, 5], device=DEV)
    accepted, want = plain.speculative_step(last, torch.full((3, 4), 7, dtype=torch.int64, device=DEV), emb, head, DraftVerifier(3, 4, V),
                                            n_drafts=torch.zeros(3, dtype=torch.int32, device=DEV))
    assert accepted.tolist() == [0, 0, 0]
    drafts = torch.tensor([[-1] * 4, [V, 1 << 40, -(1 << 40), 3], [-1, 2, 3, 4]], device=DEV)
    accepted, out = padded.speculative_step(last, drafts, emb, head, DraftVerifier(3, 4, V),
                                            n_drafts=torch.tensor([0, 4, 4], dtype=torch.int32, device=DEV))
    assert accepted.tolist() == [0, 0, 0] and torch.equal(out, want)
    assert padded.cache.lengths.tolist() == [1, 1, 1]
    # a next token that is none: the step runs, for its sequence and the others
    last = out[:, 0].clone()
    accepted, ref = plain.speculative_step(last, drafts, emb, head, DraftVerifier(3, 4, V))
    last[1] = -1
    accepted, out = padded.speculative_step(last, drafts, emb, head, DraftVerifier(3, 4, V))
    assert torch.equal(out[[0, 2]], ref[[0, 2]])
    torch.cuda.synchronize()


def test_the_example_ends_where_no_token_can_be_drawn(monkeypatch):
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_speculative_decode.py"
    spec = importlib.util.spec_from_file_location("paged_speculative_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)

    class Nothing:
        def __init__(self, batch, drafts, vocab, device="cuda"):
            pass

        def __call__(self, logits, drafts, **random):
            return (torch.zeros(logits.shape[0], dtype=torch.int32, device=DEV),
                    torch.full(logits.shape[:2], -1, dtype=torch.int64, device=DEV))

    monkeypatch.setattr(mod, "DraftVerifier", Nothing)
    with pytest.raises(RuntimeError, match="no token"):
        mod.main(["--layers", "1", "--prompt", "40", "--budget", "32", "--tokens", "4", "--vocab", "100"])
