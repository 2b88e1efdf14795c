"""GPU test of greedy speculation, every sequence for itself: the tokens are
those of one-token steps, except from a place on where the target's two best
logits nearly tie.

A near tie: the linears of one row and of several round apart by 2e-3 of the
hidden state's length (``tests/test_gpu_paged_decoder.py``); spread evenly over
its dimensions that moves the difference of two logits, with a standard
deviation of 2e-3 * |h| * |w| * sqrt(2 / hidden); six of them.
"""

import math

import pytest
import torch
import torch.nn.functional as F

from tests.test_gpu_paged_weights import _decoder

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.mark.parametrize("batch,drafts", [(2, 3), (4, 6), (3, 1)])
def test_greedy_speculation_of_every_sequence(batch, drafts):
    from turbopress_b200.speculative import DraftVerifier
    V, n = 500, 24
    g = torch.Generator(device=DEV).manual_seed(batch)
    emb = torch.randn(V, 1024, generator=g, device=DEV).half()
    head = (emb * 0.05).contiguous()
    first = torch.randint(0, V, (batch,), generator=g, device=DEV)
    dec, last = _decoder(batch), first
    plain, gaps = [], []
    for _ in range(n):
        h = dec.step(F.embedding(last[:, None], emb))
        dec.cache.advance(1)
        logits = F.linear(h, head)[:, 0].float()
        top = logits.topk(2, -1).values
        bound = 6 * 2e-3 * float(h.float().norm(dim=-1).max()) * float(head.float().norm(dim=-1).max()) * math.sqrt(2 / 1024)
        last = logits.argmax(-1)
        plain.append(last.tolist())
        gaps.append([float(t[0] - t[1]) > bound for t in top])
    plain, gaps = list(zip(*plain)), list(zip(*gaps))
    dec, last = _decoder(batch), first
    ver, said, most = DraftVerifier(batch, drafts, V), [[] for _ in range(batch)], 0
    while min(map(len, said)) < n - drafts - 1:
        # the right continuation, with a wrong token at a place that varies (or none)
        guess = [[plain[b][min(len(said[b]) + i, n - 1)] for i in range(drafts)] for b in range(batch)]
        for b in range(batch):
            at = (len(said[b]) + b) % (drafts + 1)
            if at < drafts:
                guess[b][at] = (guess[b][at] + 1 + b) % V
        accepted, out = dec.speculative_step(last, torch.tensor(guess, device=DEV), emb, head, ver)
        last = out.gather(1, accepted.long()[:, None])[:, 0].contiguous()
        for b in range(batch):
            k = int(accepted[b])
            assert (out[b, :k + 1] >= 0).all() and (out[b, k + 1:] == -1).all()
            said[b] += out[b, :k + 1].tolist()
            most = max(most, k)
            if len(said[b]) > n:  # (its continuation is not known any more)
                said[b] = said[b][:n]
    assert most >= 1  # drafts were taken
    assert dec.cache.next_pos.tolist() == dec.cache.lengths.tolist()
    for b in range(batch):
        for i, (got, want) in enumerate(zip(said[b], plain[b])):
            if got != want:
                assert not gaps[b][i], (b, i)  # a near tie; what follows is another text
                break
