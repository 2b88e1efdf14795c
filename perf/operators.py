"""The serving operators around a paged key-value cache: plain forms and cases.

Four operators, as a decode server calls them layer by layer and step by step:

* ``rope``: rotary positions of a step's (or a prompt's) queries and keys, with
  the per-head RMS norm before them where the model has one, and the append of
  keys and values into the sequences' pages;
* ``attn``: attention of each sequence's new token(s) over its pages, with the
  slots' accumulated attention weights where the cache is bounded;
* ``evict``: keep the slots of largest accumulated weight, and the first and
  latest positions, by moving survivors into the holes of the kept range;
* ``verify``: accept or replace drafted tokens by the target's logits from given
  random numbers.

``run`` computes the plain form with elementary torch operations in 32 bits, or,
with ``own`` set, makes a user's calls of ``turbopress_b200``.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"


# -- cases -------------------------------------------------------------------

def listed():
    return [
        # one sequence's decode step in the 32 / 8-head decoder: latency counts
        dict(name="rope_step", op="rope", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, scaling="default", dtype="fp16", paged=True, page=16, start=1024, norm=True, inverse=False),
        # a prompt's chunk for the 64 / 8-head decoder, positions scaled for a long context
        dict(name="rope_prompt", op="rope", batch=1, tokens=8192, q_heads=64, kv_heads=8, dim=128, rot=128,
             interleaved=False, scaling="llama3", dtype="bf16", paged=True, page=64, start=8192, norm=False, inverse=False),
        # part of each head in the interleaved layout, an odd count of tokens, views of one projection's output
        dict(name="rope_part", op="rope", batch=3, tokens=333, q_heads=16, kv_heads=8, dim=128, rot=64,
             interleaved=True, scaling="yarn", dtype="fp16", paged=False, page=16, start=100000, norm=False, inverse=False),
        # one sequence over a 1024-token cache: the smallest real call
        dict(name="attn_one", op="attn", batch=1, tokens=1, q_heads=32, kv_heads=8, dim=128, page=16, length=1024,
             ragged=False, dtype="fp16", weights=False, lse=False),
        # one long context
        dict(name="attn_long", op="attn", batch=1, tokens=1, q_heads=64, kv_heads=8, dim=128, page=64, length=131071,
             ragged=False, dtype="bf16", weights=False, lse=True),
        # a server's batch with lengths from a hundred to 8000 tokens
        dict(name="attn_ragged", op="attn", batch=64, tokens=1, q_heads=32, kv_heads=8, dim=128, page=16, length=8000,
             ragged=True, dtype="fp16", weights=False, lse=False),
        # four drafted tokens and the one before them, in a bounded cache that counts attention weights
        dict(name="attn_draft", op="attn", batch=8, tokens=5, q_heads=16, kv_heads=8, dim=128, page=32, length=4099,
             ragged=True, dtype="fp16", weights=True, lse=False),
        # a bounded cache in steady state: sixty-four steps past its budget
        dict(name="evict_step", op="evict", batch=8, kv_heads=8, dim=128, page=16, length=1088, ragged=False,
             budget=1024, recent=128, sinks=4, dtype="fp16"),
        # prompts cut down to their budget
        dict(name="evict_prompt", op="evict", batch=16, kv_heads=8, dim=128, page=64, length=16384, ragged=True,
             budget=2048, recent=256, sinks=4, dtype="bf16"),
        # greedy drafts of one sequence
        dict(name="verify_greedy", op="verify", batch=1, drafts=4, vocab=151936, dtype="fp32", probs=False,
             temperature=0.0, ragged=False),
        # a batch that samples, with the draft model's probabilities
        dict(name="verify_sample", op="verify", batch=32, drafts=7, vocab=128256, dtype="fp16", probs=True,
             temperature=0.8, ragged=False),
        # a small odd vocabulary, drafts looked up in the prompt, some sequences with fewer of them
        dict(name="verify_odd", op="verify", batch=5, drafts=3, vocab=5003, dtype="bf16", probs=False,
             temperature=1.0, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "attn", "evict", "verify"))
    heads, kv = rng.choice(((32, 8), (16, 8), (64, 8), (8, 8), (12, 4), (7, 1)))
    dim = rng.choice((64, 128, 128, 128, 96, 80))
    page = rng.choice((8, 16, 32, 64))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "rope":
        tokens = _log(rng, 1, 4000)
        return dict(op=op, batch=max(1, min(_log(rng, 1, 64), 8000 // tokens)), tokens=tokens, q_heads=heads, kv_heads=kv,
                    dim=dim, rot=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.4,
                    scaling=rng.choice(("default", "linear", "llama3", "yarn")), dtype=dtype, paged=rng.random() < 0.6,
                    page=page, start=_log(rng, 1, 4000), norm=rng.random() < 0.4, inverse=rng.random() < 0.2)
    if op == "attn":
        length = _log(rng, 1, 40000)
        return dict(op=op, batch=max(1, min(_log(rng, 1, 96), 100000 // length)), tokens=rng.choice((1, 1, 1, 2, 5, 8)),
                    q_heads=heads, kv_heads=kv, dim=dim, page=page, length=length, ragged=rng.random() < 0.6, dtype=dtype,
                    weights=rng.random() < 0.35, lse=rng.random() < 0.35)
    if op == "evict":
        length = _log(rng, 40, 16000)
        budget = max(16, int(length * rng.uniform(0.05, 0.98)))
        return dict(op=op, batch=max(1, min(_log(rng, 1, 24), 100000 // length)), kv_heads=kv, dim=dim, page=page, length=length,
                    ragged=rng.random() < 0.5, budget=budget, recent=budget // rng.choice((4, 8, 16)), sinks=rng.choice((0, 4)),
                    dtype=dtype)
    vocab = rng.choice((151936, 128256, 5003, _log(rng, 100, 150000)))
    return dict(op=op, batch=max(1, min(_log(rng, 1, 64), 4000000 // vocab)), drafts=rng.randint(1, 8), vocab=vocab,
                dtype=rng.choice(("fp16", "bf16", "fp32")), probs=rng.random() < 0.5, temperature=rng.choice((0.0, 0.7, 1.0)),
                ragged=rng.random() < 0.4)


# -- inputs ------------------------------------------------------------------

def _lengths(case):
    """Tokens in each sequence's cache: equal ones, or spread evenly over their logarithm."""
    n, top = case["batch"], case.get("length", case.get("start"))
    if not case.get("ragged") or n == 1:
        return [top] * n
    low = max(1.0, top / 80)
    return [int(math.ceil(low * (top / low) ** (b / (n - 1)) - 1e-6)) for b in range(n)]


def _frequencies(case):
    """Inverse frequencies of the rotary pairs (32 bits) and the factor on cos and sin."""
    rot, kind = case["rot"], case["scaling"]
    inv = 1.0 / (500000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))
    scale = 1.0
    if kind == "linear":
        inv = inv / 4.0
    elif kind == "llama3":  # long waves stretched by 8, short ones kept, a ramp between
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / 8.0)
    elif kind == "yarn":
        turns = 32768 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / 4.0)
        scale = 0.1 * math.log(4.0) + 1.0
    return inv.float(), scale


def _table(lens, page, generator):
    """A page of its own for every `page` tokens of each sequence, in random order; -1 where a sequence has no page."""
    counts = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(counts), generator=generator, device=DEV).int()
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, sum(counts)


def _pages(pages, case, generator, dtype, std=1.0):
    x = torch.empty(pages, case["kv_heads"], case["page"], case["dim"], dtype=dtype, device=DEV)
    return x.normal_(0.0, std, generator=generator)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    dt = DTYPES[case["dtype"]]
    make = {"rope": _prepare_rope, "attn": _prepare_attn, "evict": _prepare_evict, "verify": _prepare_verify}
    make[case["op"]](s, case, g, dt)
    if own:  # the handles that a program keeps
        _handles(s, case)
    return s


def _shuffled(case, g):
    """The sequences' lengths in an order that the seed gives."""
    lens = _lengths(case)
    order = torch.randperm(len(lens), generator=g, device=DEV).tolist()
    return [lens[i] for i in order]


def _prepare_rope(s, case, g, dt):
    b, t, hq, hk, d = (case[k] for k in ("batch", "tokens", "q_heads", "kv_heads", "dim"))
    start = [max(0, case["start"] - 7 * i) for i in range(b)]
    if case["paged"]:  # the projections' outputs
        s["q"] = torch.randn(b, t, hq, d, generator=g, device=DEV).to(dt)
        s["k"] = torch.randn(b, t, hk, d, generator=g, device=DEV).to(dt)
        s["v"] = torch.randn(b, t, hk, d, generator=g, device=DEV).to(dt)
        s["table"], n = _table([x + t for x in start], case["page"], g)
        s["k_pages"] = torch.zeros(n, hk, case["page"], d, dtype=dt, device=DEV)
        s["v_pages"] = torch.zeros_like(s["k_pages"])
    else:  # views of one fused projection's output
        fused = torch.randn(b, t, (hq + 2 * hk) * d, generator=g, device=DEV).to(dt)
        s["q"] = fused[..., :hq * d].unflatten(-1, (hq, d))
        s["k"] = fused[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    s["lengths"] = torch.tensor(start, dtype=torch.int32, device=DEV)
    s["positions"] = s["lengths"].long()[:, None] + torch.arange(t, device=DEV)
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(dt)
        s["k_norm"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(dt)
    s["inv_freq"], s["scale"] = _frequencies(case)
    # the plain form's table of cos and sin over the positions in use, rounded to 32 bits from 64
    s["first"] = min(start)
    angle = torch.arange(s["first"], max(start) + t, device=DEV, dtype=torch.float64)[:, None] * s["inv_freq"].to(DEV).double()
    s["cos"], s["sin"] = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()


def _prepare_attn(s, case, g, dt):
    b, t, hq, hk, d = (case[k] for k in ("batch", "tokens", "q_heads", "kv_heads", "dim"))
    before = _shuffled(case, g)  # tokens before the step's own
    s["total"] = [n + t for n in before]
    s["table"], n = _table(s["total"], case["page"], g)
    s["lengths"] = torch.tensor(before, dtype=torch.int32, device=DEV)
    s["q"] = torch.randn(b, t, hq, d, generator=g, device=DEV).mul_(1.5).to(dt)
    s["k_pages"], s["v_pages"] = _pages(n, case, g, dt), _pages(n, case, g, dt)
    # a page's slots past its sequence's end hold what memory held before
    last = s["table"].gather(1, torch.tensor([[(x - 1) // case["page"]] for x in s["total"]], device=DEV))[:, 0].long()
    used = torch.tensor([(x - 1) % case["page"] + 1 for x in s["total"]], device=DEV)
    stale = (torch.arange(case["page"], device=DEV) >= used[:, None])[:, None, :, None]
    for x in (s["k_pages"], s["v_pages"]):
        x[last] = x[last].masked_fill(stale, float("nan"))
    s["scores"] = None
    if case["weights"]:
        s["scores"] = torch.rand(b, hk, s["table"].shape[1] * case["page"], generator=g, device=DEV).mul_(4.0 / max(s["total"]))


def _prepare_evict(s, case, g, dt):
    b, hk = case["batch"], case["kv_heads"]
    lens = _shuffled(case, g)
    s["table"], n = _table(lens, case["page"], g)
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["k_pages"], s["v_pages"] = _pages(n, case, g, dt), _pages(n, case, g, dt)
    cap = s["table"].shape[1] * case["page"]
    # few slots hold most of the weight; earlier evictions have left the positions out of order
    s["scores"] = torch.empty(b, hk, cap, device=DEV).exponential_(generator=g).pow_(3).mul_(0.05)
    slot = torch.arange(cap, device=DEV)
    order = torch.rand(b, hk, cap, generator=g, device=DEV).masked_fill_(slot >= s["lengths"][:, None, None], 2.0).argsort(-1)
    s["positions"] = torch.where(slot < s["lengths"][:, None, None], order, -1).int()
    s["next_pos"] = s["lengths"].clone()


def _prepare_verify(s, case, g, dt):
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    target = torch.randn(b, k + 1, v, generator=g, device=DEV).mul_(2.5)
    draft = target[:, :k] + 0.7 * torch.randn(b, k, v, generator=g, device=DEV)
    s["logits"] = target.to(dt)
    s["temperature"] = torch.full((b,), case["temperature"], device=DEV)
    if case["temperature"] > 0 and b > 2:
        s["temperature"][1] = 0.0  # one greedy sequence among those that sample
    noise = torch.empty(b, k, v, device=DEV).exponential_(generator=g)
    q = torch.softmax(draft / (case["temperature"] or 1.0), -1)
    if case["probs"]:
        s["drafts"], s["probs"] = (q / noise).argmax(-1), q
    else:
        s["drafts"], s["probs"] = draft.argmax(-1), None
    s["uniforms"] = torch.rand(b, k, generator=g, device=DEV)
    s["noise"] = torch.empty(b, v, device=DEV).exponential_(generator=g)
    s["counts"] = torch.randint(0, k + 1, (b,), generator=g, device=DEV, dtype=torch.int32) if case["ragged"] else None


def _handles(s, case):
    from turbopress_b200.paged import PagedKVCache
    from turbopress_b200.rotary import Rotary
    from turbopress_b200.speculative import DraftVerifier
    if case["op"] == "rope":
        s["rotary"] = Rotary(case["dim"], s["inv_freq"], interleaved=case["interleaved"], scale=s["scale"], device=DEV)
    if case["op"] == "verify":
        s["verifier"] = DraftVerifier(case["batch"], case["drafts"], case["vocab"], device=DEV)
    elif case["op"] != "rope" or case["paged"]:
        places = s["positions"] if case["op"] == "evict" else None
        s["cache"] = PagedKVCache.from_tensors(s["k_pages"], s["v_pages"], s["table"], s["lengths"], scores=s.get("scores"),
                                               positions=places, next_pos=s.get("next_pos"))


# -- one pass ----------------------------------------------------------------

def run(state):
    forms = _OWN if own else _PLAIN
    return forms[state["case"]["op"]](state, state["case"])


def _own_rope(s, case):
    if case["paged"]:
        q = s["cache"].append(s["rotary"], s["q"], s["k"], s["v"], s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                              inverse=case["inverse"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    q, k = s["rotary"](s["q"], s["k"], s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"], inverse=case["inverse"])
    return {"q": q, "k": k}


def _own_attn(s, case):
    got = s["cache"].attend(s["q"], accumulate=case["weights"], return_lse=case["lse"])
    out, lse = got if case["lse"] else (got, None)
    return {"out": out, "lse": lse, "scores": s["scores"]}


def _own_evict(s, case):
    lengths, scores, positions = s["cache"].evict_slots(case["budget"], recent=case["recent"], sinks=case["sinks"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lengths": lengths, "scores": scores, "positions": positions}


def _own_verify(s, case):
    accepted, tokens = s["verifier"](s["logits"], s["drafts"], uniforms=s["uniforms"], noise=s["noise"], draft_probs=s["probs"],
                                     temperature=s["temperature"], n_drafts=s["counts"])
    return {"accepted": accepted, "tokens": tokens}


def _plain_rope(s, case):
    at = s["positions"] - s["first"]
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    if case["inverse"]:
        sin = -sin
    rot = case["rot"]

    def turn(x, weight):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        part = y[..., :rot]
        if case["interleaved"]:
            a, c = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * cos - c * sin, c * cos + a * sin), -1).flatten(-2)
        else:
            a, c = part[..., :rot // 2], part[..., rot // 2:]
            part = torch.cat((a * cos - c * sin, c * cos + a * sin), -1)
        return torch.cat((part, y[..., rot:]), -1).to(x.dtype)

    q, k = turn(s["q"], s["q_norm"]), turn(s["k"], s["k_norm"])
    if not case["paged"]:
        return {"q": q, "k": k}
    slot = s["lengths"].long()[:, None] + torch.arange(case["tokens"], device=DEV)
    page = s["table"].long().gather(1, slot // case["page"])
    s["k_pages"][page, :, slot % case["page"]] = k
    s["v_pages"][page, :, slot % case["page"]] = s["v"]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attn(s, case):
    b, t, hq, hk, d = (case[k] for k in ("batch", "tokens", "q_heads", "kv_heads", "dim"))
    at = s["table"].long().clamp(min=0)
    k = s["k_pages"][at].float().transpose(1, 2).reshape(b, hk, -1, d)  # [b, kv, slots, d]
    v = s["v_pages"][at].float().transpose(1, 2).reshape(b, hk, -1, d)
    slot = torch.arange(k.shape[2], device=DEV)
    seen = slot < (s["lengths"][:, None] + torch.arange(1, t + 1, device=DEV))[:, :, None]  # [b, t, slots]
    held = (slot < s["lengths"][:, None] + t)[:, None, :, None]
    v = torch.where(held, v, 0.0)
    q = s["q"].float().reshape(b, t, hk, hq // hk, d).transpose(1, 2).reshape(b, hk, -1, d)  # rows: token, head of the group
    logit = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    seen = seen[:, None, :, None].expand(b, 1, t, hq // hk, -1).reshape(b, 1, -1, k.shape[2])
    logit = torch.where(seen, logit, float("-inf"))
    top = logit.amax(-1, keepdim=True)
    p = torch.exp(logit - top)
    total = p.sum(-1, keepdim=True)
    out = (torch.matmul(p, v) / total).reshape(b, hk, t, -1, d).transpose(1, 2).reshape(b, t, hq, d).to(s["q"].dtype)
    lse = None
    if case["lse"]:
        lse = (top + total.log()).reshape(b, hk, t, -1).transpose(1, 2).reshape(b, t, hq)
    if case["weights"]:
        s["scores"] += (p / total).sum(2)
    return {"out": out, "lse": lse, "scores": s["scores"]}


def _plain_evict(s, case):
    budget, cap = case["budget"], s["scores"].shape[-1]
    lens = s["lengths"][:, None, None]
    slot = torch.arange(cap, device=DEV)
    pos = s["positions"]
    guarded = (pos < case["sinks"]) | (pos >= s["next_pos"][:, None, None] - case["recent"])
    key = torch.where(guarded, float("inf"), s["scores"])
    key = torch.where(slot < lens, key, float("-inf"))
    order = key.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order[..., :budget], True) & (slot < lens)
    hole, late = ~kept & (slot < budget) & (slot < lens), kept & (slot >= budget)
    # the n-th survivor above the budget goes to the n-th hole below it
    where_hole = torch.nonzero(hole)
    where_late = torch.nonzero(late)
    b, h, to, come = where_hole[:, 0], where_hole[:, 1], where_hole[:, 2], where_late[:, 2]
    page = s["table"].long()
    src, dst = page[b, come // case["page"]], page[b, to // case["page"]]
    for x in (s["k_pages"], s["v_pages"]):
        x[dst, h, to % case["page"]] = x[src, h, come % case["page"]]
    scores, places = s["scores"].clone(), pos.clone()
    scores[b, h, to], places[b, h, to] = s["scores"][b, h, come], pos[b, h, come]
    count = s["lengths"].clamp(max=budget)
    live = slot < count[:, None, None]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "lengths": count,
            "scores": torch.where(live, scores, 0.0), "positions": torch.where(live, places, -1)}


def _plain_verify(s, case):
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    greedy = s["temperature"] == 0
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    token = torch.arange(v, device=DEV)
    best = torch.where(x == top, token, v).amin(-1)  # [b, k + 1]
    p = torch.exp((x - top) / torch.where(greedy, 1.0, s["temperature"])[:, None, None])
    p = p / p.sum(-1, keepdim=True)
    at = s["drafts"][:, :, None]
    chance = 1.0 if s["probs"] is None else s["probs"].gather(2, at)[..., 0]
    fine = s["uniforms"] * chance < p[:, :k].gather(2, at)[..., 0]
    fine = torch.where(greedy[:, None], best[:, :k] == s["drafts"], fine)
    count = torch.full((b,), k, device=DEV) if s["counts"] is None else s["counts"].long()
    fine &= torch.arange(k, device=DEV) < count[:, None]
    accepted = fine.int().cumprod(-1).sum(-1)
    row = torch.arange(b, device=DEV)
    goal = p[row, accepted]  # [b, v]
    used = accepted.clamp(max=k - 1)
    drafted = (token == s["drafts"][row, used][:, None]).float() if s["probs"] is None else s["probs"][row, used]
    rest = torch.where((accepted < count)[:, None], (goal - drafted).clamp(min=0), goal)
    rest = torch.where(rest.amax(-1, keepdim=True) > 0, rest, goal)
    race = rest / s["noise"]
    drawn = torch.where(race == race.amax(-1, keepdim=True), token, v).amin(-1)
    final = torch.where(greedy, best[row, accepted], drawn)
    place = torch.arange(k + 1, device=DEV)
    padded = torch.cat((s["drafts"], final[:, None]), 1)
    tokens = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], final[:, None], -1))
    return {"accepted": accepted.int(), "tokens": tokens}


_PLAIN = {"rope": _plain_rope, "attn": _plain_attn, "evict": _plain_evict, "verify": _plain_verify}
_OWN = {"rope": _own_rope, "attn": _own_attn, "evict": _own_evict, "verify": _own_verify}


# -- the definition in 64 bits -------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    return {"rope": _exact_rope, "attn": _exact_attn, "evict": _exact_evict, "verify": _exact_verify}[case["op"]](s, case)


def _exact_rope(s, case):
    rot = case["rot"]
    angle = s["positions"].double()[..., None] * s["inv_freq"].to(DEV).double()
    turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if case["inverse"] else angle)[:, :, None]

    def one(x, weight):
        y = x.double()
        if weight is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * weight.double()
        pairs = y[..., :rot].unflatten(-1, (rot // 2, 2)) if case["interleaved"] else y[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, y[..., rot:]), -1)

    q, k = one(s["q"], s["q_norm"]), one(s["k"], s["k_norm"])
    if not case["paged"]:
        return {"q": q, "k": k}
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    for b, first in enumerate(s["lengths"].tolist()):
        i = torch.arange(case["tokens"], device=DEV)
        page, off = s["table"][b].long()[(first + i) // case["page"]], (first + i) % case["page"]
        kp[page, :, off], vp[page, :, off] = k[b], s["v"][b].double()
    return {"q": q, "k_pages": kp, "v_pages": vp}


def _exact_attn(s, case):
    t, hk, d = case["tokens"], case["kv_heads"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:3], dtype=torch.float64, device=DEV)
    scores = s["scores"].double() if case["weights"] else None
    group = case["q_heads"] // hk
    for b, n in enumerate(s["total"]):
        pages = s["table"][b, :-(-n // case["page"])].long()
        for h in range(hk):
            k = s["k_pages"][pages, h].reshape(-1, d)[:n].double()
            v = s["v_pages"][pages, h].reshape(-1, d)[:n].double()
            for i in range(t):
                m = n - t + i + 1
                z = s["q"][b, i, h * group:(h + 1) * group].double() @ k[:m].T / math.sqrt(d)
                lse[b, i, h * group:(h + 1) * group] = torch.logsumexp(z, -1)
                w = torch.softmax(z, -1)
                out[b, i, h * group:(h + 1) * group] = w @ v[:m]
                if scores is not None:
                    scores[b, h, :m] += w.sum(0)
    return {"out": out, "lse": lse if case["lse"] else None, "scores": scores}


def _exact_evict(s, case):
    got = _plain_evict(s, case)  # moves and comparisons alone: nothing is rounded
    return {k: x.double() if x.is_floating_point() else x for k, x in got.items()}


def _exact_verify(s, case):
    k = case["drafts"]
    counts = [k] * case["batch"] if s["counts"] is None else s["counts"].tolist()
    accepted, rows = [], []
    for b in range(case["batch"]):
        heat = float(s["temperature"][b])
        x = s["logits"][b].double()
        drafts, said = s["drafts"][b].tolist(), []
        for i in range(counts[b] + 1):
            p = torch.softmax(x[i] / heat, -1) if heat else (torch.arange(x.shape[-1], device=DEV) == int((x[i] == x[i].max()).nonzero()[0])).double()
            q = None
            if i < counts[b]:
                q = torch.zeros_like(p)
                if s["probs"] is not None and heat:
                    q = s["probs"][b, i].double()
                else:
                    q[drafts[i]] = 1.0
                sure = p[drafts[i]] > 0 if not heat else s["uniforms"][b, i].double() * q[drafts[i]] < p[drafts[i]]
                if bool(sure):
                    said.append(drafts[i])
                    continue
            rest = p if q is None or not heat else (p - q).clamp(min=0)
            rest = rest if float(rest.max()) > 0 else p
            said.append(int((rest / (s["noise"][b].double() if heat else 1.0)).argmax()))
            break
        accepted.append(len(said) - 1)
        rows.append(said + [-1] * (k + 1 - len(said)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32, device=DEV), "tokens": torch.tensor(rows, device=DEV)}


# -- work --------------------------------------------------------------------

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    if case["op"] == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        sampled = 0 if case["temperature"] == 0 else b - (1 if b > 2 else 0)
        return {"bytes": b * (k + 1) * v * size + sampled * v * (4 + (4 if case["probs"] else 0)), "flops": 4 * b * (k + 1) * v}
    d, hk = case["dim"], case["kv_heads"]
    if case["op"] == "rope":
        n, hq = case["batch"] * case["tokens"], case["q_heads"]
        heads = hq + hk * (2 if case["paged"] else 1)
        return {"bytes": 2 * n * heads * d * 2, "flops": 3 * n * (hq + hk) * case["rot"]}
    lens = _lengths(case)
    if case["op"] == "attn":
        total, rows, hq = sum(lens) + len(lens) * case["tokens"], case["batch"] * case["tokens"], case["q_heads"]
        return {"bytes": total * hk * d * 4 + 4 * rows * hq * d + (8 * total * hk if case["weights"] else 0),
                "flops": 4 * total * hq * d * case["tokens"]}
    budget, page = case["budget"], case["page"]
    cap = max(-(-n // page) for n in lens) * page
    guard = case["recent"] + case["sinks"]
    # positions and weights are in random order: a kept slot lies above the budget with probability 1 - budget / length
    moved = sum(budget * (1 - budget / n) for n in lens if n > budget)
    return {"bytes": hk * (8 * sum(lens) + 8 * cap * len(lens) + moved * d * 2 * 2 * 2), "flops": hk * sum(lens) * (2 if guard else 1)}
