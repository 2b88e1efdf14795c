"""Plain 64-bit restatements of the paged-cache operators, for the tests.

Tensors may be on any device; everything is computed in float64 (moves and
comparisons excepted) with loops over sequences and heads.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor


def rotate(x: Tensor, positions: Tensor, inv_freq: Tensor, scale: float = 1.0, interleaved: bool = False,
           inverse: bool = False, weight: Tensor | None = None, eps: float = 1e-6) -> Tensor:
    """x [..., heads, dim] at positions [...]; float64."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = inv_freq.numel()
    # the angle as a sum of two exact products (20 bits of the position at a time)
    f = inv_freq.to(x.device).double()
    low = positions & ((1 << 20) - 1)
    a, b = (positions - low).double()[..., None, None] * f, low.double()[..., None, None] * f
    c = (a.cos() * b.cos() - a.sin() * b.sin()) * scale
    s = (a.sin() * b.cos() + a.cos() * b.sin()) * scale * (-1 if inverse else 1)
    out = y.clone()
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    return out


def slots_of(pages: Tensor, table_row: Tensor, n: int) -> tuple[Tensor, Tensor]:
    """Rows [n, kv_heads, dim] of the first n slots of a sequence and which of
    them have a page; pages [num_pages, kv_heads, page_size, dim]."""
    ps = pages.shape[2]
    s = torch.arange(n, device=pages.device)
    ids = table_row.long()[s // ps]
    ok = (ids >= 0) & (ids < pages.shape[0])
    rows = pages[ids.clamp(0, pages.shape[0] - 1), :, s % ps]
    return rows, ok


def attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, scale: float | None = None):
    """(out, lse, weights [batch, kv_heads, capacity]) in float64."""
    B, T, Hq, D = q.shape
    Hk = k_pages.shape[1]
    g = Hq // Hk
    cap = table.shape[1] * k_pages.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    weights = torch.zeros(B, Hk, cap, dtype=torch.float64, device=q.device)
    for b in range(B):
        if int(lengths[b]) < 0:
            continue
        for j in range(T):
            n = min(int(lengths[b]) + j + 1, cap)
            k, ok = slots_of(k_pages, table[b], n)
            v, _ = slots_of(v_pages, table[b], n)
            k, v, at = k[ok].double(), v[ok].double(), torch.nonzero(ok)[:, 0]
            if not len(at):
                continue
            for h in range(Hq):
                s = (k[:, h // g] @ q[b, j, h].double()) * scale
                lse[b, j, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                out[b, j, h] = p @ v[:, h // g]
                weights[b, h // g, at] += p
    return out, lse, weights


def evict(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, next_pos: Tensor, scores: Tensor,
          positions: Tensor, budget: int, recent: int = 0, sinks: int = 0):
    """(k_pages, v_pages, lengths, scores, positions) after the eviction."""
    kp, vp, ns, npos = k_pages.clone(), v_pages.clone(), torch.zeros_like(scores), torch.full_like(positions, -1)
    cap = scores.shape[2]
    ps = k_pages.shape[2]
    new_len = []
    for b in range(len(lengths)):
        n = max(0, min(int(lengths[b]), cap))
        new_len.append(min(int(lengths[b]), budget, cap))
        for h in range(scores.shape[1]):
            pos, sc = positions[b, h].tolist(), scores[b, h].tolist()

            def key(i):
                guarded = pos[i] < sinks or pos[i] >= int(next_pos[b]) - recent
                return (0 if guarded else 1, 0 if math.isnan(sc[i]) else 1, 0.0 if math.isnan(sc[i]) or guarded else -sc[i], i)

            kept = sorted(sorted(range(n), key=key)[:budget])
            live = set(kept)
            holes = [i for i in range(min(n, budget)) if i not in live]
            late = [i for i in kept if i >= budget]
            assert len(holes) == len(late)
            place = {i: i for i in kept if i < budget}
            place.update(dict(zip(late, holes)))
            for i, to in place.items():
                ns[b, h, to], npos[b, h, to] = scores[b, h, i], positions[b, h, i]
                if i != to:
                    src, dst = int(table[b, i // ps]), int(table[b, to // ps])
                    if 0 <= src < len(kp) and 0 <= dst < len(kp):
                        kp[dst, h, to % ps], vp[dst, h, to % ps] = k_pages[src, h, i % ps], v_pages[src, h, i % ps]
    return kp, vp, torch.tensor(new_len, dtype=torch.int32, device=lengths.device), ns, npos


def verify(logits: Tensor, drafts: Tensor, uniforms, noise, probs, temperature, counts):
    """(accepted, tokens, margin): margin is how far the nearest comparison was
    from equality (relative), infinite for whole-number ones."""
    B, rows, V = logits.shape
    accepted, tokens, margin = [], [], math.inf
    for b in range(B):
        t = 0.0 if temperature is None else float(temperature[b])
        n = rows - 1 if counts is None else max(0, min(int(counts[b]), rows - 1))
        said = []
        for r in range(n + 1):
            x = logits[b, r].double()
            if t <= 0:
                nan = torch.isnan(x)
                best = int(torch.nonzero(nan if nan.any() else x == x.max())[0, 0])
                if r < n and int(drafts[b, r]) == best:
                    said.append(best)
                    continue
                said.append(best)
                break
            p = torch.softmax(x / t, -1)
            q = None
            if r < n:
                d = int(drafts[b, r])
                q = torch.zeros_like(p)
                if probs is not None:
                    q = probs[b, r].double()
                elif 0 <= d < V:
                    q[d] = 1.0
                if 0 <= d < V:
                    need, have = float(uniforms[b, r]) * float(q[d]), float(p[d])
                    if max(need, have) > 0:
                        margin = min(margin, abs(need - have) / max(need, have))
                    if need < have:
                        said.append(d)
                        continue
            rest = p if q is None else (p - q).clamp(min=0)
            if not float(rest.max()) > 0:
                rest = p
            race = rest / noise[b].double()
            race = torch.where(rest > 0, race, 0.0)
            if not float(race.max()) > 0:
                said.append(-1)
                break
            top = race.topk(min(2, V)).values
            if len(top) > 1 and math.isfinite(float(top[0])):
                margin = min(margin, float((top[0] - top[1]) / top[0]))
            said.append(int(torch.nonzero(race == race.max())[0, 0]))
            break
        accepted.append(len(said) - 1)
        tokens.append(said + [-1] * (rows - len(said)))
    return (torch.tensor(accepted, dtype=torch.int32, device=logits.device), torch.tensor(tokens, device=logits.device), margin)
