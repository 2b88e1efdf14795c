"""GPU tests of the operators together: ``PagedDecoder`` against the torch
restatement of the reference model's forward and against itself (tokens at
once or one by one), and the example's loop."""

import numpy as np
import pytest
import torch

from tests.conftest import GOLDEN
from tests.step_reference import reference_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _decoder(batch, page=16, pages=8, qk_norm=True, seed=3, track=False):
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.paged_decoder import PagedDecoder
    from turbopress_b200.synthetic import step_config, synthetic_decoder
    cfg = dict(name="test", layers=2, hidden=1024, inter=2048, q_heads=16, kv_heads=8, head_dim=128,
               rope_theta=1_000_000.0, qk_norm=qk_norm)
    with np.load(GOLDEN / "codebooks.npz") as f:
        cbs = {3: torch.from_numpy(f["opt_b3_s64"])}
    layers, fnorm = synthetic_decoder(cfg, [3, 3], cbs, DEV, seed=seed)
    cache = PagedKVCache(batch, 8, 128, batch * pages, page, pages, layers=2, track_weights=track)
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache.block_table.copy_(torch.randperm(batch * pages, generator=g, device=DEV).view(batch, pages))
    return PagedDecoder(layers, step_config(cfg), fnorm, cache), layers, cfg, fnorm, g


@pytest.mark.parametrize("qk_norm", [True, False])
def test_matches_the_reference_forward(qk_norm):
    """Token by token against the restated fp16 forward (rel L2 1e-2, as the
    fused decode step is held to: the two round activations at other places)."""
    from turbopress_b200.step import DecodeStep
    from turbopress_b200.synthetic import step_config
    dec, layers, cfg, fnorm, g = _decoder(2, qk_norm=qk_norm)
    step = DecodeStep(layers, step_config(cfg), fnorm, batch=2, max_tokens=64)
    kc, vc = step.k_cache.clone(), step.v_cache.clone()
    for pos in range(20):
        x = torch.randn(2, 1024, device=DEV, generator=g).half()
        ref, _ = reference_step(step, x, pos, kc, vc)
        out = dec.step(x[:, None])[:, 0]
        dec.cache.advance(1)
        rel = float((out.float() - ref.float()).norm() / ref.float().norm())
        assert rel < 1e-2, (pos, rel)
    dec.cache.status()
    assert dec.cache.lengths.tolist() == [20, 20] == dec.cache.next_pos.tolist()


def test_tokens_at_once_or_one_by_one():
    """A chunk of tokens gives what its tokens give one by one (rel L2 2e-3:
    another linear kernel above eight rows)."""
    dec, *_, g = _decoder(2)
    x = torch.randn(2, 30, 1024, device=DEV, generator=g).half()
    whole = dec.step(x)
    parts = []
    for c in range(0, 30, 7):
        parts.append(dec.step(x[:, c:c + 7]))
        dec.cache.advance(min(7, 30 - c))
    single = torch.cat(parts, 1)
    rel = float((whole.float() - single.float()).norm() / single.float().norm())
    assert rel < 2e-3, rel


def test_rejected_tokens_leave_no_trace():
    """Advancing by fewer tokens than were appended: the next step overwrites the rest."""
    dec, *_, g = _decoder(1)
    x = torch.randn(1, 12, 1024, device=DEV, generator=g).half()
    junk = torch.randn(1, 6, 1024, device=DEV, generator=g).half()
    dec.step(x[:, :8])
    dec.cache.advance(8)
    dec.step(torch.cat((x[:, 8:9], junk[:, :4]), 1))  # four rejected drafts
    dec.cache.advance(1)
    with_junk = dec.step(x[:, 9:12])
    clean, *_ = _decoder(1)
    clean.step(x[:, :8])
    clean.cache.advance(8)
    clean.step(x[:, 8:9])
    clean.cache.advance(1)
    want = clean.step(x[:, 9:12])
    rel = float((with_junk.float() - want.float()).norm() / want.float().norm())
    assert rel < 2e-3, rel


def test_greedy_speculation_continues_as_greedy():
    """At temperature 0 drafts change the speed alone: the tokens are those of
    one-token steps (up to a near tie of two logits)."""
    from turbopress_b200.speculative import DraftVerifier
    torch.manual_seed(0)
    V = 500
    emb = torch.randn(V, 1024, device=DEV).half()
    head = (emb * 0.05).contiguous()
    dec, *_ = _decoder(2)
    ver = DraftVerifier(2, 0, V)
    none = torch.zeros(2, 0, dtype=torch.int64, device=DEV)
    last = torch.tensor([3, 4], device=DEV)
    plain = []
    for _ in range(20):
        _, out = dec.speculative_step(last, none, emb, head, ver)
        last = out[:, 0].contiguous()
        plain.append(last.tolist())
    plain = list(zip(*plain))
    dec, *_ = _decoder(2)
    ver = DraftVerifier(2, 3, V)
    last = torch.tensor([3, 4], device=DEV)
    said = [[], []]
    wrong = 0
    while min(map(len, said)) < 16:
        # the right continuation, with a wrong token at a place that varies
        drafts = [[plain[b][(len(said[b]) + i) % 20] for i in range(3)] for b in range(2)]
        for b in range(2):
            drafts[b][len(said[b]) % 3] = (drafts[b][len(said[b]) % 3] + (len(said[b]) % 2)) % V
        accepted, out = dec.speculative_step(last, torch.tensor(drafts, device=DEV), emb, head, ver)
        last = out.gather(1, accepted.long()[:, None])[:, 0].contiguous()
        for b in range(2):
            said[b] += out[b, :int(accepted[b]) + 1].tolist()
    for b in range(2):
        n = min(16, len(said[b]))
        wrong += said[b][:n] != list(plain[b][:n])
    assert wrong <= 1  # (one sequence may have met a near tie)


@pytest.mark.parametrize("temperature", [0.8, 0.0])
def test_example_runs(temperature, capsys):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_speculative_decode.py"
    spec = importlib.util.spec_from_file_location("paged_speculative_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    got = mod.main(["--layers", "2", "--prompt", "300", "--chunk", "128", "--budget", "200", "--tokens", "24", "--vocab", "600",
                    "--temperature", str(temperature)])
    assert all(len(s) >= 324 and all(0 <= t < 600 for t in s) for s in got["said"])
    assert all(n <= got["capacity"] for n in got["lengths"])
    # positions go on counting past what was evicted
    assert got["next_pos"] == [len(s) - 1 for s in got["said"]]
    assert "rounds" in capsys.readouterr().out


def test_refusals():
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.paged_decoder import PagedDecoder
    dec, layers, cfg, fnorm, _ = _decoder(1)
    for cache in (PagedKVCache(1, 8, 128, 8, 16, 8), PagedKVCache(1, 4, 128, 8, 16, 8, layers=2),
                  PagedKVCache(1, 8, 128, 8, 16, 8, layers=2, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            PagedDecoder(layers, dec.cfg, fnorm, cache)
