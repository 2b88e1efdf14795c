"""A packed decoder over a paged cache: any number of tokens per sequence in a step.

``DecodeStep`` runs one token of up to eight sequences in one launch over
contiguous caches.  ``PagedDecoder`` runs the same decoder layers
(``LayerWeights``: seven ``PackedTCQLinear`` and the norms) call by call over a
``PagedKVCache``: prompts in chunks, drafted tokens, sequences of any lengths,
caches held to a budget.

    decoder = PagedDecoder(layers, cfg, final_norm, cache)
    hidden = decoder.step(embeddings)          # [batch, tokens, hidden] -> final norm's output
    cache.advance(tokens)                      # or as many as were accepted

``speculative_step`` is one round of drafting: target over the last token and
its drafts, verification, and the cache cut back to what was accepted.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import Tensor

from .paged import PagedKVCache
from .rotary import Rotary
from .speculative import DraftVerifier
from .step import LayerWeights, StepConfig


def _rms_norm(x: Tensor, w: Tensor, eps: float) -> Tensor:
    """The models' RMS norm: fp32 inside, rounded before the weight."""
    x32 = x.float()
    return w * (x32 * torch.rsqrt(x32.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype)


class PagedDecoder:
    """Decoder layers over a paged cache (fp16, as the packed linears)."""

    def __init__(self, layers: list[LayerWeights], cfg: StepConfig, final_norm: Tensor, cache: PagedKVCache,
                 rotary: Rotary | None = None) -> None:
        """``rotary`` defaults to the configuration's plain one (it holds no
        scaling: ``Rotary.from_config(config)`` for a checkpoint that has one)."""
        if cache.layers != len(layers) or (cache.kv_heads, cache.head_dim) != (cfg.kv_heads, cfg.head_dim):
            raise ValueError("the cache's layers, kv_heads and head_dim must be the decoder's")
        if cache.dtype != torch.float16:
            raise ValueError("packed decoders run in fp16")
        self.layers, self.cfg, self.cache = layers, cfg, cache
        self.rotary = Rotary(cfg.head_dim, theta=cfg.rope_theta, device=cache.device) if rotary is None else rotary

        def on_device(w: Tensor | None) -> Tensor | None:
            return None if w is None else w.to(device=cache.device, dtype=torch.float16).contiguous()

        self.final_norm = on_device(final_norm)
        self.norms = [tuple(on_device(w) for w in (lw.ln1, lw.ln2, lw.q_norm, lw.k_norm)) for lw in layers]

    def step(self, embeddings: Tensor, accumulate: bool = False, held: list[tuple[Tensor, Tensor]] | None = None) -> Tensor:
        """[batch, tokens, hidden] input embeddings of each sequence's next
        tokens -> the final norm's output for each.  The tokens are in the
        cache behind ``lengths`` afterwards; ``cache.advance`` counts them.
        ``accumulate``: add to the cache's attention weights.  ``held``: takes
        each layer's queries and log-sum-exp, for ``cache.add_weights`` once it
        is known which of the tokens stay."""
        cfg, cache = self.cfg, self.cache
        B, T, _ = embeddings.shape
        h = embeddings.to(torch.float16)
        for i, (lw, (ln1, ln2, q_norm, k_norm)) in enumerate(zip(self.layers, self.norms)):
            x = _rms_norm(h, ln1, cfg.rms_eps)
            q = lw.q(x).view(B, T, cfg.q_heads, cfg.head_dim)
            k = lw.k(x).view(B, T, cfg.kv_heads, cfg.head_dim)
            v = lw.v(x).view(B, T, cfg.kv_heads, cfg.head_dim)
            q = cache.append(self.rotary, q, k, v, layer=i, q_norm=q_norm, k_norm=k_norm, eps=cfg.rms_eps)
            if held is None:
                out = cache.attend(q, layer=i, accumulate=accumulate)
            else:
                out, lse = cache.attend(q, layer=i, accumulate=accumulate, return_lse=True)
                held.append((q, lse))
            h = h + lw.o(out.view(B, T, -1))
            x = _rms_norm(h, ln2, cfg.rms_eps)
            h = h + lw.down(F.silu(lw.gate(x)) * lw.up(x))
        return _rms_norm(h, self.final_norm, cfg.rms_eps)

    def speculative_step(self, tokens: Tensor, drafts: Tensor, embedding: Tensor, lm_head: Tensor, verifier: DraftVerifier, *,
                         accumulate: bool = False, **random) -> tuple[Tensor, Tensor]:
        """One round: ``tokens`` int64 [batch] (chosen, not yet in the cache)
        and ``drafts`` int64 [batch, drafts] after them through the decoder,
        the drafts verified against the logits (``random``: uniforms, noise,
        draft_probs, temperature, n_drafts as ``DraftVerifier`` takes them).
        Returns (accepted [batch], tokens [batch, drafts + 1]); the cache holds
        the token and the accepted drafts, and with ``accumulate`` their
        attention weights.  Ids outside the vocabulary are looked up as its
        nearest: such a draft (padding behind n_drafts, say) is rejected, and a
        next token of -1, of a row without any probability, is for the caller
        to end the sequence at."""
        ids = torch.cat((tokens[:, None], drafts), 1).clamp_(0, embedding.shape[0] - 1)
        held: list[tuple[Tensor, Tensor]] | None = [] if accumulate else None
        hidden = self.step(F.embedding(ids, embedding), held=held)
        accepted, out = verifier(F.linear(hidden, lm_head), drafts, **random)
        stay = accepted + 1
        for i, (q, lse) in enumerate(held or ()):
            self.cache.add_weights(q, lse, stay, layer=i)
        self.cache.advance(stay)
        return accepted, out
