"""Verification of drafted tokens: ``tp_verify_drafts`` behind a small class.

The reference's decode loops take one greedy token per step
(scripts/run_packed.py:160-190).  With drafts -- from a smaller packed model,
or looked up in the prompt -- a step runs the target over several tokens at
once (``PagedKVCache.append`` / ``attend`` with ``tokens`` > 1) and
``DraftVerifier`` decides how many of them stand, so that what comes out is
distributed as the target's own tokens (or, at temperature 0, is its greedy
continuation).

    verify = DraftVerifier(batch, drafts, vocab)
    accepted, tokens = verify(logits, draft_tokens, uniforms=u, noise=e, temperature=t)
    cache.advance(accepted + 1)                   # rejected tokens drop out of the cache

Random numbers are the caller's: ``uniforms`` in [0, 1) and ``noise`` from the
unit exponential distribution, so a run can be repeated.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from . import _abi

MAX_DRAFTS = 63


class _VerifyArgs(ctypes.Structure):
    """Mirror of ``tp_verify_args``."""

    _fields_ = [("logits", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64)] + [
        (nm, ctypes.c_void_p) for nm in ("draft_tokens", "draft_probs", "uniforms", "noise", "temperature", "counts",
                                         "accepted", "tokens")] + [
        (nm, ctypes.c_int32) for nm in ("batch", "drafts", "vocab", "dtype")]


class DraftVerifier:
    """Accepts or replaces drafted tokens by the target's logits; holds the
    workspace for up to ``batch`` sequences of ``drafts`` drafts (one verifier
    per stream)."""

    def __init__(self, batch: int, drafts: int, vocab: int, device="cuda") -> None:
        self.batch, self.drafts, self.vocab = batch, drafts, vocab
        need = _abi.lib().tp_verify_workspace_bytes(batch, drafts, vocab)
        if need < 0:
            _abi.check(-need, "DraftVerifier")
        self.workspace = torch.zeros(need, dtype=torch.uint8, device=device)
        self.device = self.workspace.device
        _abi.require_cuda(self.workspace)
        self._plans: dict[tuple, tuple[_VerifyArgs, Tensor, Tensor]] = {}

    def __call__(self, logits: Tensor, draft_tokens: Tensor, *, uniforms: Tensor | None = None, noise: Tensor | None = None,
                 draft_probs: Tensor | None = None, temperature: Tensor | None = None,
                 n_drafts: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """logits [batch, drafts + 1, vocab] (fp16 / bf16 / fp32, contiguous
        elements), draft_tokens int64 [batch, drafts], uniforms fp32 [batch,
        drafts], noise fp32 [batch, vocab], draft_probs fp32 [batch, drafts,
        vocab] or None (drafts taken without sampling), temperature fp32
        [batch] (0: greedy; None: all greedy), n_drafts int32 [batch] (drafts
        in use; None: all).  Returns accepted int32 [batch] and tokens int64
        [batch, drafts + 1]: the accepted drafts, the next token, then -1."""
        key = (_abi.meta(logits), _abi.meta(draft_tokens), _abi.meta(uniforms), _abi.meta(noise), _abi.meta(draft_probs),
               _abi.meta(temperature), _abi.meta(n_drafts))
        plan = self._plans.get(key)
        if plan is None:
            plan = self._checked(logits, draft_tokens, uniforms, noise, draft_probs, temperature, n_drafts)
            if len(self._plans) >= 256:
                self._plans.clear()
            self._plans[key] = plan
        template, like_accepted, like_tokens = plan
        accepted, tokens = torch.empty_like(like_accepted), torch.empty_like(like_tokens)
        a = _VerifyArgs.from_buffer_copy(template)
        a.logits, a.draft_tokens, a.accepted, a.tokens = (logits.data_ptr(), draft_tokens.data_ptr(), accepted.data_ptr(),
                                                          tokens.data_ptr())
        if temperature is not None:
            a.temperature, a.noise = temperature.data_ptr(), noise.data_ptr()
            if uniforms is not None:
                a.uniforms = uniforms.data_ptr()
            if draft_probs is not None:
                a.draft_probs = draft_probs.data_ptr()
        if n_drafts is not None:
            a.counts = n_drafts.data_ptr()
        _abi.launch(_abi.lib().tp_verify_drafts, "verify_drafts", self.device.index, ctypes.addressof(a),
                    self.workspace.data_ptr(), self.workspace.numel())
        return accepted, tokens

    def _checked(self, logits: Tensor, draft_tokens: Tensor, uniforms: Tensor | None, noise: Tensor | None,
                 draft_probs: Tensor | None, temperature: Tensor | None, n_drafts: Tensor | None) -> tuple[_VerifyArgs, Tensor, Tensor]:
        """Checks a call by what its key holds; the sizes and strides of its
        arguments, and tensors like its outputs."""
        if logits.dim() != 3:
            raise ValueError(f"logits must be [batch, drafts + 1, vocab], got {tuple(logits.shape)}")
        B, rows, V = logits.shape
        K = rows - 1
        if not (1 <= B <= self.batch and 0 <= K <= self.drafts and V == self.vocab):
            raise ValueError(f"logits {tuple(logits.shape)} do not fit a verifier of ({self.batch}, {self.drafts} + 1, {self.vocab})")
        if logits.stride(2) != 1:
            raise ValueError("logits rows must be contiguous")
        sampled = temperature is not None
        if sampled and (noise is None or (K and uniforms is None)):
            raise ValueError("sampling needs uniforms and noise")
        for t, shape, dt, nm in ((draft_tokens, (B, K), torch.int64, "draft_tokens"), (uniforms, (B, K), torch.float32, "uniforms"),
                                 (noise, (B, V), torch.float32, "noise"), (draft_probs, (B, K, V), torch.float32, "draft_probs"),
                                 (temperature, (B,), torch.float32, "temperature"), (n_drafts, (B,), torch.int32, "n_drafts")):
            if t is not None and (t.shape != shape or t.dtype != dt or t.device != self.device or not t.is_contiguous()):
                raise ValueError(f"{nm} must be a contiguous {dt} tensor {shape} on {self.device}")
        if logits.device != self.device:
            raise ValueError(f"logits must be on {self.device}")
        return (_VerifyArgs(batch_stride=logits.stride(0), row_stride=logits.stride(1), batch=B, drafts=K, vocab=V,
                            dtype=_abi.dtype_code(logits.dtype)),
                torch.empty(B, dtype=torch.int32, device=self.device), torch.empty(B, rows, dtype=torch.int64, device=self.device))
