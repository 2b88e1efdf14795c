"""Speculative decoding of a packed decoder over a bounded paged cache.

A random-init Qwen3-shaped decoder (a few packed 3-bit layers) reads a prompt
in chunks, then decodes with drafts looked up in what was said before, while
each sequence's cache is held to a budget of slots by accumulated attention
weight:

    python examples/paged_speculative_decode.py [--layers 4] [--tokens 64] [--temperature 0.8]

Per layer and step: packed linears, ``PagedKVCache.append`` (head norms, rotary
positions, pages), ``attend``; per step ``DraftVerifier``; every ``--stride``
steps ``evict``.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch
import torch.nn.functional as F

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from turbopress_b200.paged import PagedKVCache  # noqa: E402
from turbopress_b200.paged_decoder import PagedDecoder  # noqa: E402
from turbopress_b200.speculative import DraftVerifier  # noqa: E402
from turbopress_b200.synthetic import QWEN3_0_6B, step_config, synthetic_decoder  # noqa: E402


def look_up(said: list[int], drafts: int) -> list[int]:
    """The tokens that followed the last earlier occurrence of the final two
    (repeated to `drafts` of them; zeros where there is none)."""
    for i in range(len(said) - 3, 0, -1):
        if said[i - 1:i + 1] == said[-2:]:
            found = said[i + 1:i + 1 + drafts]
            return (found * drafts)[:drafts]
    return [0] * drafts


def main(argv: list[str] | None = None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=4096)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--chunk", type=int, default=256)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--budget", type=int, default=512)
    ap.add_argument("--stride", type=int, default=8)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device())
    cfg = {**QWEN3_0_6B, "layers": a.layers}
    with np.load(ROOT / "tests" / "golden" / "codebooks.npz") as f:
        codebooks = {3: torch.from_numpy(f["opt_b3_s64"])}
    layers, final_norm = synthetic_decoder(cfg, [3] * a.layers, codebooks, dev, seed=a.seed)
    g = torch.Generator(device=dev).manual_seed(a.seed)
    embedding = torch.randn(a.vocab, cfg["hidden"], generator=g, device=dev).half()
    lm_head = (embedding * 0.05).contiguous()

    page = 16
    most = max(a.prompt, a.budget) + a.stride * (a.drafts + 1) + a.drafts + 1
    pages = -(-most // page)
    cache = PagedKVCache(a.batch, cfg["kv_heads"], cfg["head_dim"], a.batch * pages, page, pages, layers=a.layers,
                         track_weights=True, device=dev)
    cache.block_table.copy_(torch.randperm(a.batch * pages, generator=g, device=dev).view(a.batch, pages))
    decoder = PagedDecoder(layers, step_config(cfg), final_norm, cache)
    verifier = DraftVerifier(a.batch, a.drafts, a.vocab, device=dev)
    temperature = torch.full((a.batch,), a.temperature, device=dev)

    prompt = torch.randint(0, a.vocab, (a.batch, a.prompt), generator=g, device=dev)
    for c in range(0, a.prompt - 1, a.chunk):  # all but the last prompt token, which the first round takes
        ids = prompt[:, c:min(c + a.chunk, a.prompt - 1)]
        decoder.step(F.embedding(ids, embedding), accumulate=True)
        cache.advance(ids.shape[1])
    cache.evict(a.budget, recent=a.budget // 4, sinks=4)

    said = prompt.tolist()
    last = prompt[:, -1].contiguous()
    rounds = accepted_total = 0
    while min(len(s) for s in said) < a.prompt + a.tokens:
        drafts = torch.tensor([look_up(s, a.drafts) for s in said], device=dev)
        accepted, out = decoder.speculative_step(
            last, drafts, embedding, lm_head, verifier, accumulate=True, temperature=temperature,
            uniforms=torch.rand(a.batch, a.drafts, generator=g, device=dev),
            noise=torch.empty(a.batch, a.vocab, device=dev).exponential_(generator=g))
        last = out.gather(1, accepted.long()[:, None])[:, 0].contiguous()
        for s, row, n in zip(said, out.tolist(), accepted.tolist()):
            if row[n] < 0:
                raise RuntimeError("the logits leave no token to draw (not finite?)")
            s += row[:n + 1]
            accepted_total += n
        rounds += 1
        if rounds % a.stride == 0:
            cache.evict(a.budget, recent=a.budget // 4, sinks=4)
    cache.status()
    print(f"{rounds} rounds, {sum(len(s) - a.prompt for s in said) / (rounds * a.batch):.2f} tokens per sequence and round, "
          f"cache lengths {cache.lengths.tolist()}, next positions {cache.next_pos.tolist()}")
    return dict(rounds=rounds, said=said, accepted=accepted_total, lengths=cache.lengths.tolist(), next_pos=cache.next_pos.tolist(),
                capacity=cache.capacity)


if __name__ == "__main__":
    main()
