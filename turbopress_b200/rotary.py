"""Rotary positions: ``tp_rotary`` behind a small class.

The decode step's rotary embedding is the plain one (half layout, the whole
head, unscaled frequencies).  ``Rotary`` covers the layouts and scalings that
other checkpoints and long contexts need -- half or interleaved pairs, part of
the head, linear / llama3 / yarn scaled frequencies -- for any number of
tokens, with the per-head RMS norm that Qwen3 applies before it.

    rotary = Rotary.from_config(model.config)            # a Hugging Face config
    q, k = rotary(q, k, positions)                        # [..., heads, head_dim], int64 [...]
    q = cache.append(rotary, q, k, v)                     # the same, k and v into a PagedKVCache

Angles are exact modulo one turn for every position (a 64-bit phase, not a
32-bit product); arithmetic is fp32 with one rounding to the tensors' dtype.  No
gradients are recorded; ``inverse`` is the rotation's.
"""

from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import torch
from torch import Tensor

from . import _abi

# 2^192 / (2 pi), from 60 digits of pi
_TURNS = int(2 ** 191 / Fraction("3.14159265358979323846264338327950288419716939937510582097494"))
SCALINGS = ("default", "linear", "llama3", "yarn")


class _RotaryArgs(ctypes.Structure):
    """Mirror of ``tp_rotary_args``."""

    _fields_ = [(nm, ctypes.c_void_p) for nm in ("q", "k", "v", "q_out", "k_out", "positions", "base", "freq", "q_norm",
                                                 "k_norm")] + [
        (nm, ctypes.c_int64) for nm in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride",
                                        "v_token_stride", "v_head_stride", "tokens")] + [
        (nm, ctypes.c_int32) for nm in ("seq", "q_heads", "kv_heads", "head_dim", "rot_dim", "dtype", "interleaved",
                                        "inverse")] + [("scale", ctypes.c_float), ("eps", ctypes.c_float)]


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: dict | None = None) -> tuple[Tensor, float]:
    """(inverse frequencies fp32 [rot_dim/2], factor on cos and sin).

    ``scaling`` holds a Hugging Face config's rope parameters: ``rope_type``
    one of ``SCALINGS``, ``factor`` and what the type needs beside it
    (``original_max_position_embeddings``; ``low_freq_factor`` /
    ``high_freq_factor`` for llama3; ``beta_fast`` / ``beta_slow`` /
    ``attention_factor`` for yarn)."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be a positive even number, got {rot_dim}")
    inv = 1.0 / (theta ** (torch.arange(0, rot_dim, 2, dtype=torch.int64).to(dtype=torch.float) / rot_dim))
    p = scaling or {}
    kind = p.get("rope_type", p.get("type", "default"))
    if kind not in SCALINGS:
        raise ValueError(f"unsupported rope type {kind!r} (one of {SCALINGS})")
    if kind == "default":
        return inv, 1.0
    factor = float(p["factor"])
    if kind == "linear":  # every position divided by the factor
        return inv / factor, 1.0
    # llama3 and yarn: waves that turn often within the original context stay
    # as they are, those that do not complete a few turns are stretched by the
    # factor, and a linear ramp joins the two
    original = float(p["original_max_position_embeddings"])
    if kind == "llama3":
        low, high = float(p["low_freq_factor"]), float(p["high_freq_factor"])
        turns = original * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return inv * keep + inv / factor * (1 - keep), 1.0

    # yarn: the ramp is over the pair's index, between the pairs that make
    # beta_fast and beta_slow turns in the original context
    def pair_of(turns: float) -> float:
        return rot_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

    first, last = pair_of(float(p.get("beta_fast") or 32)), pair_of(float(p.get("beta_slow") or 1))
    if p.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rot_dim - 1)
    ramp = ((torch.arange(rot_dim // 2, dtype=torch.float) - first) / max(last - first, 0.001)).clamp(0, 1)

    def temperature(scale: float, m: float = 1.0) -> float:
        return 0.1 * m * math.log(scale) + 1.0 if scale > 1 else 1.0

    attention = p.get("attention_factor")
    if attention is None:
        m, m_all = p.get("mscale"), p.get("mscale_all_dim")
        attention = temperature(factor, m) / temperature(factor, m_all) if m and m_all else temperature(factor)
    return inv * (1 - ramp) + inv / factor * ramp, float(attention)


def _turn_word(f: float) -> int:
    """round(f 2^64 / (2 pi)) mod 2^64 of an fp32 value, in whole numbers."""
    mantissa, exponent = math.frexp(f)
    shift = 152 - exponent  # f = n 2^(exponent - 24)
    return ((int(mantissa * 2 ** 24) * _TURNS + (1 << (shift - 1))) >> shift) % 2 ** 64


class Rotary:
    """Rotary positions of one model: its frequencies, laid out once."""

    def __init__(self, head_dim: int, inv_freq: Tensor | None = None, *, theta: float = 10000.0,
                 scaling: dict | None = None, rot_dim: int | None = None, interleaved: bool = False,
                 scale: float | None = None, device="cuda") -> None:
        if inv_freq is None:
            inv_freq, factor = rope_frequencies(head_dim if rot_dim is None else rot_dim, theta, scaling)
            scale = factor if scale is None else scale
        if inv_freq.dim() != 1 or (rot_dim is not None and 2 * inv_freq.numel() != rot_dim):
            raise ValueError("inv_freq must be 1-D with rot_dim / 2 entries")
        self.head_dim, self.rot_dim = int(head_dim), 2 * inv_freq.numel()
        if not 2 <= self.rot_dim <= self.head_dim <= 256 or self.head_dim % 2:
            raise ValueError(f"need an even head_dim <= 256 and rot_dim <= head_dim, got {head_dim} and {self.rot_dim}")
        self.interleaved, self.scale = bool(interleaved), 1.0 if scale is None else float(scale)
        self.inv_freq = inv_freq.detach().to(device="cpu", dtype=torch.float32)
        if not torch.isfinite(self.inv_freq).all():
            raise ValueError("inv_freq must be finite")
        # turns per position as 64-bit fractions of a turn; whole turns drop out
        words = [_turn_word(f) for f in self.inv_freq.tolist()]
        self.freq = torch.tensor([w - 2 ** 64 if w >= 2 ** 63 else w for w in words], dtype=torch.int64).to(device)
        self.device = self.freq.device
        self._plans: dict[tuple, _RotaryArgs] = {}

    @classmethod
    def from_config(cls, config, device="cuda", interleaved: bool = False) -> "Rotary":
        """From a Hugging Face decoder config (its theta, scaling and partial
        factor).  A config with parameters for each kind of layer has a Rotary
        for each of them, and is refused here."""
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        p = getattr(config, "rope_parameters", None) or getattr(config, "rope_scaling", None) or {}
        kinds = [k for k, v in p.items() if isinstance(v, dict)]
        if kinds:
            raise ValueError(f"the config has rope parameters for each kind of layer ({', '.join(kinds)}): make a Rotary of each, "
                             "Rotary(head_dim, theta=..., scaling=...)")
        theta = float(p.get("rope_theta") or getattr(config, "rope_theta", None) or 10000.0)
        part = float(p.get("partial_rotary_factor") or getattr(config, "partial_rotary_factor", None) or 1.0)
        if p and "original_max_position_embeddings" not in p and getattr(config, "max_position_embeddings", None):
            p = {**p, "original_max_position_embeddings": config.max_position_embeddings}
        return cls(head_dim, theta=theta, scaling=p, rot_dim=int(head_dim * part), interleaved=interleaved, device=device)

    # -- arguments shared with PagedKVCache.append ------------------------------
    def _args(self, plans: dict, adapt, q: Tensor, k: Tensor, v: Tensor | None, positions: Tensor | None,
              q_norm: Tensor | None, k_norm: Tensor | None, eps: float, inverse: bool) -> tuple[_RotaryArgs, Tensor, tuple]:
        """The call's arguments without k's destination, the queries' output and
        the tensors to keep until the launch.  ``plans`` holds the checked part
        by what the checks depend on; ``adapt(plan, q, k, v)`` completes a new one."""
        key = (_abi.meta(q), _abi.meta(k), _abi.meta(v), _abi.meta(positions), _abi.meta(q_norm), _abi.meta(k_norm))
        plan = plans.get(key)
        if plan is None:
            plan = self._checked(q, k, v, positions, q_norm, k_norm)
            if plan is None:  # not views of [tokens, heads, head_dim]
                return self._args(plans, adapt, q.contiguous(), k.contiguous(), None if v is None else v.contiguous(), positions,
                                  q_norm, k_norm, eps, inverse)
            if adapt is not None:
                adapt(plan, q, k, v)
            if len(plans) >= 256:
                plans.clear()
            plans[key] = plan
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a = _RotaryArgs.from_buffer_copy(plan)
        a.q, a.k, a.q_out, a.inverse, a.eps = q.data_ptr(), k.data_ptr(), out.data_ptr(), inverse, eps
        if v is not None:
            a.v = v.data_ptr()
        if positions is not None:
            if positions.dtype is not torch.int64 or not positions.is_contiguous():
                positions = positions.to(torch.int64).contiguous()
            a.positions = positions.data_ptr()
        if q_norm is not None:
            a.q_norm = q_norm.data_ptr()
        if k_norm is not None:
            a.k_norm = k_norm.data_ptr()
        return a, out, (q, k, v, positions)

    def _checked(self, q: Tensor, k: Tensor, v: Tensor | None, positions: Tensor | None, q_norm: Tensor | None,
                 k_norm: Tensor | None) -> _RotaryArgs | None:
        """The part of the arguments that shapes, strides and dtypes decide;
        None where q, k or v is not a view of [tokens, heads, head_dim]."""
        hd = self.head_dim
        if q.dim() < 2 or k.dim() != q.dim() or q.shape[-1] != hd or k.shape[-1] != hd or q.shape[:-2] != k.shape[:-2]:
            raise ValueError(f"q and k must be [..., heads, {hd}] over the same tokens, got {tuple(q.shape)} and {tuple(k.shape)}")
        for t in (q, k, v):
            if t is not None and (t.dtype != q.dtype or t.device != self.device):
                raise ValueError("q, k and v must share one dtype and be on the frequencies' CUDA device")
        if v is not None and v.shape != k.shape:
            raise ValueError(f"v must have k's shape {tuple(k.shape)}, got {tuple(v.shape)}")
        if positions is not None and (positions.shape != q.shape[:-2] or positions.device != self.device):
            raise ValueError(f"positions must be {tuple(q.shape[:-2])} on {self.device}, got {tuple(positions.shape)}")
        for w in (q_norm, k_norm):
            if w is not None and (w.shape != (hd,) or w.dtype != q.dtype or w.device != self.device or not w.is_contiguous()):
                raise ValueError(f"norm weights must be contiguous [{hd}] tensors of the queries' dtype and device")
        a = _RotaryArgs(freq=self.freq.data_ptr(), seq=1, q_heads=q.shape[-2], kv_heads=k.shape[-2], head_dim=hd,
                        rot_dim=self.rot_dim, dtype=_abi.dtype_code(q.dtype), interleaved=self.interleaved, scale=self.scale)
        for nm, t in (("q", q), ("k", k), ("v", v)):
            if t is None:
                continue
            try:
                flat = t.view(-1, t.shape[-2], hd) if t.numel() else t.reshape(0, t.shape[-2], hd)
            except RuntimeError:
                return None
            if flat.stride(2) != 1:
                return None
            setattr(a, nm + "_token_stride", flat.stride(0))
            setattr(a, nm + "_head_stride", flat.stride(1))
        a.tokens = math.prod(q.shape[:-2])
        return a

    def __call__(self, q: Tensor, k: Tensor, positions: Tensor, *, q_norm: Tensor | None = None,
                 k_norm: Tensor | None = None, eps: float = 1e-6, inverse: bool = False) -> tuple[Tensor, Tensor]:
        """q [..., q_heads, head_dim] and k [..., kv_heads, head_dim] at integer
        ``positions`` [...] -> the rotated pair (new contiguous tensors), on the
        current stream.  ``q_norm`` / ``k_norm`` [head_dim]: RMS norm of each
        head before it.  ``inverse`` turns back, which is also the gradient of
        the rotation."""
        if positions is None:
            raise ValueError("positions are needed")
        a, q_out, keep = self._args(self._plans, None, q, k, None, positions, q_norm, k_norm, eps, inverse)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        a.k_out = k_out.data_ptr()
        _abi.launch(_abi.lib().tp_rotary, "rotary", self.device.index, ctypes.addressof(a), None)
        return q_out, k_out
