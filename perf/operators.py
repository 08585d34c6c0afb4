"""Performance cases of the operators around the projections of a decode step on one MI355X.

A decoding program goes through them in this order: rotary positions written
into a paged key-value cache, attention of the new tokens over that cache
(adding up, where it evicts, what weight each cached token gets), and, after
the output head, probabilities from logits and the verification of drafted
tokens; when a sequence has used up its budget, eviction by the weights added up.

`run` makes one pass: where `own` is false in elementary torch operations in 32
bits, where it is true through this framework's entry points.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"f32": (torch.float32, 4, 0), "f16": (torch.float16, 2, 1), "bf16": (torch.bfloat16, 2, 30)}
VOCAB = 151936
FIXED = 36  # fractional bits of the verification's fixed-point weights

_ctx = None


def _package():
    path = str(Path(__file__).resolve().parent.parent / "memory-aware-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import si_hip
    return si_hip


def _context():
    """The process's context, as a program keeps one for its lifetime."""
    global _ctx
    if _ctx is None:
        _ctx = _package().HipContext(0)
    return _ctx


def listed():
    return [
        # one token of one sequence enters the cache: the smallest call of a decode step. The q rows
        # lie beside their output gates, a quarter of each head rotates.
        {"name": "rope_token", "kind": "rope", "sequences": 1, "tokens": 1, "heads": 24,
         "kv_heads": 4, "head_dim": 256, "rotary": 64, "layout": "half", "scaling": "none",
         "theta": 1e7, "gated": True, "type": "bf16", "page": 16, "capacity": 4096},
        # chunks of four prompts, whole heads rotated in pairs, stretched for a long context
        {"name": "rope_prompt", "kind": "rope", "sequences": 4, "tokens": 2043, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rotary": 128, "layout": "interleaved",
         "scaling": "yarn", "theta": 1e6, "gated": False, "type": "f16", "page": 64,
         "capacity": 4096},
        # the next token of one short conversation: latency is most of it
        {"name": "attn_token", "kind": "attn", "sequences": 1, "tokens": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "type": "f16", "page": 16, "lo": 1021, "hi": 1021,
         "window": 0, "ragged": False, "weights": False},
        # the next token after a very long document: the cache's bytes are all of it
        {"name": "attn_long", "kind": "attn", "sequences": 1, "tokens": 1, "heads": 24,
         "kv_heads": 4, "head_dim": 256, "type": "bf16", "page": 16, "lo": 131071, "hi": 131071,
         "window": 0, "ragged": False, "weights": False},
        # drafted tokens of a few sequences of different lengths, verified in one pass
        {"name": "attn_verify", "kind": "attn", "sequences": 4, "tokens": 8, "heads": 24,
         "kv_heads": 4, "head_dim": 256, "type": "bf16", "page": 32, "lo": 700, "hi": 16001,
         "window": 0, "ragged": True, "weights": False},
        # a batch that keeps account of its tokens' weights, to evict by them; an f32 cache
        {"name": "attn_weights", "kind": "attn", "sequences": 24, "tokens": 1, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "type": "f32", "page": 64, "lo": 1, "hi": 4095,
         "window": 0, "ragged": False, "weights": True},
        # one sequence over its budget
        {"name": "evict_token", "kind": "evict", "sequences": 1, "kv_heads": 4, "head_dim": 256,
         "type": "bf16", "page": 16, "lo": 4111, "hi": 4111, "keep": 3001, "sinks": 4,
         "recent": 256},
        # a batch cut to a fraction of its length, some sequences still below the budget
        {"name": "evict_batch", "kind": "evict", "sequences": 8, "kv_heads": 8, "head_dim": 128,
         "type": "f16", "page": 64, "lo": 2000, "hi": 16384, "keep": 6144, "sinks": 16,
         "recent": 1024},
        # the logits of one sequence's drafted tokens and the one after them
        {"name": "softmax_verify", "kind": "softmax", "rows": 5, "cols": VOCAB,
         "temperature": 0.7},
        # those of a batch
        {"name": "softmax_batch", "kind": "softmax", "rows": 288, "cols": VOCAB,
         "temperature": 1.0},
        # a sequence's four drafts against the target's probabilities
        {"name": "verify_one", "kind": "verify", "sequences": 1, "drafts": 4, "vocab": VOCAB,
         "ragged": False, "certain": False},
        # a batch of up to eight drafts each
        {"name": "verify_batch", "kind": "verify", "sequences": 32, "drafts": 8, "vocab": VOCAB,
         "ragged": True, "certain": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "attn", "evict", "softmax", "verify"])
    heads, kv_heads, head_dim = rng.choice([(24, 4, 256), (32, 8, 128), (16, 16, 64), (32, 4, 128),
                                            (10, 2, 96), (8, 1, 192), (28, 4, 128), (40, 8, 80)])
    cache = {"kv_heads": kv_heads, "head_dim": head_dim, "type": rng.choice(["f32", "f16", "bf16"]),
             "page": rng.choice([8, 16, 24, 32, 64, 128])}
    if kind == "rope":
        sequences = _log(rng, 1, 32)
        tokens = _log(rng, 1, 8000 // sequences)
        rotary = rng.choice([head_dim, head_dim // 2, head_dim // 4])
        return {"kind": kind, "sequences": sequences, "tokens": tokens, "heads": heads, **cache,
                "rotary": rotary, "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "yarn"]),
                "theta": rng.choice([1e4, 1e6, 1e7]), "gated": rng.random() < 0.3,
                "capacity": tokens + _log(rng, 1, 2000)}
    if kind == "attn":
        tokens = rng.choice([1, 1, 1, rng.randint(2, 16)])
        row = kv_heads * head_dim * 2 * TYPES[cache["type"]][1]
        rows = 380_000_000 // row // (4 if tokens > 8 else 2 if tokens > 1 else 1)
        sequences = _log(rng, 1, 48)
        hi = _log(rng, 16, max(17, min(120_000, rows // sequences)))
        return {"kind": kind, "sequences": sequences, "tokens": tokens, "heads": heads, **cache,
                "lo": rng.choice([1, hi // 2 + 1, hi]), "hi": hi,
                "window": rng.choice([0, 0, 0, _log(rng, 8, 4096)]),
                "ragged": tokens > 1 and rng.random() < 0.5, "weights": rng.random() < 0.3}
    if kind == "evict":
        row = kv_heads * head_dim * 2 * TYPES[cache["type"]][1]
        sequences = _log(rng, 1, 16)
        hi = _log(rng, 600, min(32768, 300_000_000 // row // sequences))
        keep = max(64, int(hi * rng.uniform(0.2, 0.95)))
        return {"kind": kind, "sequences": sequences, **cache, "lo": rng.choice([hi // 3 + 1, hi]),
                "hi": hi, "keep": keep, "sinks": rng.randint(0, 16),
                "recent": rng.randint(0, keep // 2)}
    if kind == "softmax":
        cols = rng.choice([VOCAB, _log(rng, 1000, VOCAB)])
        return {"kind": kind, "rows": _log(rng, 1, 280), "cols": cols,
                "temperature": round(rng.uniform(0.3, 1.5), 3)}
    return {"kind": kind, "sequences": _log(rng, 1, 32), "drafts": rng.randint(1, 8),
            "vocab": rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), "ragged": rng.random() < 0.4,
            "certain": rng.random() < 0.25}


# ---- inputs ------------------------------------------------------------------

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFFFFFF)


def _normal(shape, seed, salt, scale=1.0):
    return torch.randn(shape, generator=_generator(seed, salt), device="cuda") * scale


def _spread(lo, hi, count):
    """`count` lengths from lo to hi in a fixed irregular order, hi among them."""
    return [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887) % 1.0))
            for i in range(count)]


def _lengths(case):
    return _spread(case["lo"], case["hi"], case["sequences"])


def _counts(case, most):
    """New tokens (or drafts) of each sequence: all of them, or a ragged number."""
    n = case["sequences"]
    return [most if not case["ragged"] or i % 3 == 0 else (i * 5 + 1) % (most + 1)
            for i in range(n)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(sequences, max_pages, seed, salt):
    """A page table whose sequences' pages lie all over the pool."""
    order = torch.randperm(sequences * max_pages, generator=_generator(seed, salt), device="cuda")
    return order.view(sequences, max_pages).to(torch.int32)


def _pool(pages, case, seed, salt):
    """Cached rows [pages][kv_heads][page][head_dim]."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    out = torch.empty(shape, dtype=TYPES[case["type"]][0], device="cuda")
    g = _generator(seed, salt)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for a in range(0, pages, step):
        part = out[a:a + step]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return out


def _cache(case, capacity, lengths, seed, salt, empty=False):
    max_pages = -(-capacity // case["page"])
    n = case["sequences"]
    pages = n * max_pages
    c = {"table": _pages(n, max_pages, seed, salt), "lengths": _ints(lengths)}
    if empty:
        shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
        c["keys"] = torch.zeros(shape, dtype=TYPES[case["type"]][0], device="cuda")
        c["values"] = torch.zeros_like(c["keys"])
    else:
        c["keys"] = _pool(pages, case, seed, salt + 1)
        c["values"] = _pool(pages, case, seed, salt + 2)
    return c


def _handle(case, c):
    """The framework's description of a cache, which a program makes once."""
    return _package().KvCache(
        ggml_type=TYPES[case["type"]][2], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
        page_tokens=case["page"], pages=c["keys"].shape[0], sequences=case["sequences"],
        max_pages=c["table"].shape[1], d_keys=c["keys"].data_ptr(), d_values=c["values"].data_ptr(),
        d_page_table=c["table"].data_ptr(), d_lengths=c["lengths"].data_ptr())


def _inverse_frequencies(case):
    """Radians a position for each rotated pair, in 64 bits, and the factor of cos and sin."""
    n, theta = case["rotary"], case["theta"]
    i = np.arange(n // 2, dtype=np.float64)
    inv = theta ** (-2.0 * i / n)
    if case["scaling"] == "none":
        return inv, 1.0
    factor, original = 4.0, 32768.0
    if case["scaling"] == "linear":
        return inv / factor, 1.0
    pair = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    low = max(math.floor(pair(32.0)), 0)
    high = min(math.ceil(pair(1.0)), n - 1)
    ramp = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
    return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _frequencies(case):
    """The pairs' turns a position, as 64-bit fractions of a turn."""
    inv, magnitude = _inverse_frequencies(case)
    turns = inv.astype(np.longdouble) / (2 * np.longdouble(np.pi))
    table = np.rint(turns * np.longdouble(2.0) ** 64).astype(np.uint64)
    return torch.from_numpy(table.view(np.int64)).cuda(), magnitude


def _rope_inputs(case, seed):
    b, t, d = case["sequences"], case["tokens"], case["head_dim"]
    q = _normal((b, t, case["heads"], (2 if case["gated"] else 1) * d), seed, 1)
    k = _normal((b, t, case["kv_heads"], d), seed, 2)
    v = _normal((b, t, case["kv_heads"], d), seed, 3)
    first = torch.randint(0, 120_000, (b, 1), generator=_generator(seed, 4), device="cuda")
    positions = (first + torch.arange(t, device="cuda")).to(torch.int32)
    lengths = [(case["capacity"] - t) * (i + 1) // b for i in range(b)]
    return q, k, v, positions, lengths


def _logits(rows, cols, seed, salt):
    """Rows of a head's logits: a wide bell and a few likely tokens."""
    x = _normal((rows, cols), seed, salt, 2.5)
    top = torch.randint(0, cols, (rows, 12), generator=_generator(seed, salt + 1), device="cuda")
    return x.scatter_add(1, top, _normal((rows, 12), seed, salt + 2, 2.0) + 12.0)


def _evict_weights(case, capacity, seed):
    """Weights added up over a few hundred steps: heavy tails, and tokens that nothing ever saw."""
    shape = (case["sequences"], case["kv_heads"], capacity)
    w = torch.exp(_normal(shape, seed, 5, 2.0))
    unseen = torch.rand(shape, generator=_generator(seed, 6), device="cuda") < 0.1
    return torch.where(unseen, torch.zeros_like(w), w)


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if kind == "rope":
        s["q"], s["k"], s["v"], s["positions"], lengths = _rope_inputs(case, seed)
        s["cache"] = _cache(case, case["capacity"], lengths, seed, 10)
        s["table"], s["magnitude"] = _frequencies(case)
        s["out"] = torch.empty(s["q"].shape[:3] + (case["head_dim"],), device="cuda")
    elif kind == "attn":
        b, t = case["sequences"], case["tokens"]
        # the cache already has the new tokens' rows, behind the `length` that it had before them
        s["cache"] = _cache(case, case["hi"] + t, _lengths(case), seed, 10)
        s["q"] = _normal((b, t, case["heads"], case["head_dim"]), seed, 1, 2.0)
        s["out"] = torch.empty_like(s["q"])
        s["counts"] = _ints(_counts(case, t)) if case["ragged"] else None
        s["scale"] = case["head_dim"] ** -0.5
        if case["weights"]:
            capacity = s["cache"]["table"].shape[1] * case["page"]
            s["weights"] = _normal((b, case["kv_heads"], capacity), seed, 5).abs()
    elif kind == "evict":
        s["cache"] = _cache(case, case["hi"], _lengths(case), seed, 10)
        s["to"] = _cache(case, case["keep"], [0] * case["sequences"], seed, 20, empty=True)
        capacity = s["cache"]["table"].shape[1] * case["page"]
        s["weights"] = _evict_weights(case, capacity, seed)
        to_capacity = s["to"]["table"].shape[1] * case["page"]
        shape = (case["sequences"], case["kv_heads"])
        s["to_weights"] = torch.zeros(shape + (to_capacity,), device="cuda")
        s["kept"] = torch.zeros(shape + (case["keep"],), dtype=torch.int32, device="cuda")
    elif kind == "softmax":
        s["x"] = _logits(case["rows"], case["cols"], seed, 1)
        s["out"] = torch.empty_like(s["x"])
    else:
        n, m, vocab = case["sequences"], case["drafts"], case["vocab"]
        x = _logits(n * (m + 1), vocab, seed, 1)
        y = x.view(n, m + 1, vocab)[:, :m] + _normal((n, m, vocab), seed, 7, 0.7)
        s["target"] = torch.softmax(x, 1).view(n, m + 1, vocab)
        s["draft"] = torch.softmax(y, 2)
        noise = torch.rand((n, m, vocab), generator=_generator(seed, 8), device="cuda")
        if case["certain"]:
            s["tokens"], s["draft"] = s["draft"].argmax(2).to(torch.int32), None
        else:
            s["tokens"] = (s["draft"] / -torch.log(noise.clamp(1e-12, 1 - 1e-6))).argmax(2).to(torch.int32)
        s["uniform"] = torch.rand((n, m + 1), generator=_generator(seed, 9), device="cuda")
        s["counts"] = _ints(_counts(case, m)) if case["ragged"] else None
        s["accepted"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros((n, m + 1), dtype=torch.int32, device="cuda")
    if own:  # what a program makes once and keeps: its context, its caches' handles, its scratch
        s["ctx"] = _context()
        if "cache" in s:
            s["handle"] = _handle(case, s["cache"])
        if "to" in s:
            s["to_handle"] = _handle(case, s["to"])
        if kind == "rope":
            s["rope"] = _package().Rope(layout=("half", "interleaved").index(case["layout"]),
                                        rotary_dim=case["rotary"], magnitude=s["magnitude"],
                                        d_frequencies=s["table"].data_ptr())
        if kind == "attn":
            size = s["ctx"].paged_attention_workspace(s["handle"], case["heads"], case["tokens"],
                                                      case["weights"])
            s["scratch"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return s


# ---- the operators in plain form -----------------------------------------------

def _slots(cache, page, slots):
    """Where slots [sequences][n] of each sequence lie: their pages and their rows in them."""
    return cache["table"].long().gather(1, slots // page), slots % page


def _rotate(x, phase, layout, magnitude):
    """x [b][t][h][d] with its first 2 * phase.shape[-1] values rotated; phase in turns [b][t][n]."""
    n = phase.shape[-1]
    angle = phase[:, :, None] * (2 * math.pi)
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rope(s):
    case, c = s["case"], s["cache"]
    d = case["head_dim"]
    # the fraction of a turn, exact in wrapping 64-bit integers, then 32 bits
    phase = (s["positions"].long()[:, :, None] * s["table"]).float() * 2.0 ** -64
    q = _rotate(s["q"][..., :d], phase, case["layout"], s["magnitude"])
    k = _rotate(s["k"], phase, case["layout"], s["magnitude"])
    slots = c["lengths"].long()[:, None] + torch.arange(case["tokens"], device="cuda")
    page, row = _slots(c, case["page"], slots)
    c["keys"][page, :, row] = k.to(c["keys"].dtype)
    c["values"][page, :, row] = s["v"].to(c["values"].dtype)
    return {"q": q, "keys": c["keys"], "values": c["values"]}


def _gathered(cache, what):
    """Every slot's rows of all sequences: [b][kv_heads][capacity][d] in 32 bits."""
    rows = cache[what][cache["table"].long()]
    return rows.transpose(1, 2).flatten(2, 3).float()


def _visible(case, lengths, counts, capacity):
    """[b][t][capacity]: the slots that each new token attends to."""
    t = torch.arange(case["tokens"], device="cuda")
    end = (lengths.long()[:, None] + t + 1)[:, :, None]
    slot = torch.arange(capacity, device="cuda")
    seen = slot < end
    if case["window"]:
        seen = seen & (slot >= end - case["window"])
    if counts is not None:
        seen = seen & (t < counts.long()[:, None])[:, :, None]
    return seen


def _plain_attn(s):
    case, c = s["case"], s["cache"]
    b, t, h, d = s["q"].shape
    g = h // case["kv_heads"]
    keys, values = _gathered(c, "keys"), _gathered(c, "values")
    capacity = keys.shape[2]
    seen = _visible(case, c["lengths"], s["counts"], capacity)[:, None, :, None]
    q = s["q"].view(b, t, -1, g, d).transpose(1, 2).reshape(b, -1, t * g, d)
    score = torch.matmul(q, keys.transpose(2, 3)) * s["scale"]
    score = score.view(b, -1, t, g, capacity).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.view(b, -1, t * g, capacity), values)
    out = out.view(b, -1, t, g, d).transpose(1, 2).reshape(b, t, h, d)
    if not case["weights"]:
        return out
    s["weights"] += p.sum((2, 3))
    return {"out": out, "weights": s["weights"]}


def _plain_evict(s):
    case, c, to = s["case"], s["cache"], s["to"]
    keep = case["keep"]
    weights = s["weights"]
    capacity = weights.shape[2]
    slot = torch.arange(capacity, device="cuda")
    length = c["lengths"].long()[:, None, None]
    rank = weights.masked_fill((slot < case["sinks"]) | (slot >= length - case["recent"]), math.inf)
    rank = rank.masked_fill(slot >= length, -math.inf)
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    left = length.clamp(max=keep)
    there = torch.arange(keep, device="cuda") < left
    kept = torch.sort(order.masked_fill(~there, capacity), dim=2).values
    source = kept.clamp(max=capacity - 1)
    at, row = _slots(to, case["page"], torch.arange(keep, device="cuda").expand(case["sequences"], keep))
    page = c["table"].long()[torch.arange(case["sequences"], device="cuda")[:, None, None],
                             source // case["page"]]
    head = torch.arange(case["kv_heads"], device="cuda")[:, None]
    for_head = (at[:, None], head, row[:, None])
    to["keys"][for_head] = torch.where(there[..., None], c["keys"][page, head, source % case["page"]],
                                       to["keys"][for_head])
    to["values"][for_head] = torch.where(there[..., None],
                                         c["values"][page, head, source % case["page"]],
                                         to["values"][for_head])
    s["to_weights"][:, :, :keep] = torch.where(there, weights.gather(2, source),
                                               s["to_weights"][:, :, :keep])
    to["lengths"].copy_(left.view(-1))
    s["kept"].copy_(kept.masked_fill(~there, -1))
    return _evicted(s)


def _evicted(s):
    return {"keys": s["to"]["keys"], "values": s["to"]["values"], "weights": s["to_weights"],
            "kept": s["kept"], "lengths": s["to"]["lengths"]}


def _plain_softmax(s):
    x = s["x"] / s["case"]["temperature"]
    e = torch.exp(x - x.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _plain_verify(s):
    case = s["case"]
    n, m, vocab = case["sequences"], case["drafts"], case["vocab"]
    target, draft, u = s["target"], s["draft"], s["uniform"]
    token = s["tokens"].long()[:, :, None]
    p = target[:, :m].gather(2, token)[..., 0]
    q = torch.ones_like(p) if draft is None else draft.gather(2, token)[..., 0]
    i = torch.arange(m, device="cuda")
    count = torch.full((n,), m, device="cuda") if s["counts"] is None else s["counts"].long()
    accept = (u[:, :m] * q < p) & (i < count[:, None])
    first = accept.long().cumprod(1).sum(1)
    row = target.gather(1, first[:, None, None].expand(n, 1, vocab))[:, 0]
    refused = (first < count)[:, None]
    j = first.clamp(max=m - 1)[:, None, None]
    if draft is None:
        was = torch.zeros_like(row).scatter(1, token[:, :, 0].gather(1, j[:, 0]), 1.0)
    else:
        was = draft.gather(1, j.expand(n, 1, vocab))[:, 0]
    fixed = lambda x: (x.clamp(0.0, 1.0) * 2.0 ** FIXED).long()  # noqa: E731
    rest = torch.where(refused, fixed(row - was), fixed(row))
    rest = torch.where(rest.sum(1, keepdim=True) == 0, fixed(row), rest)
    running = rest.cumsum(1)
    threshold = ((u[:, m:] * 2.0 ** 24).long() * running[:, -1:]) >> 24
    sampled = (running <= threshold).sum(1, keepdim=True)
    tokens = torch.cat([token[:, :, 0], sampled], 1)
    at = torch.arange(m + 1, device="cuda")
    out = torch.where(at < first[:, None], tokens, torch.full_like(tokens, -1))
    out = torch.where(at == first[:, None], sampled, out)
    return {"accepted": first.to(torch.int32), "tokens": out.to(torch.int32)}


# ---- one pass ------------------------------------------------------------------

def run(state):
    s = state
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"rope": _plain_rope, "attn": _plain_attn, "evict": _plain_evict,
                "softmax": _plain_softmax, "verify": _plain_verify}[kind](s)
    ctx = s["ctx"]
    if kind == "rope":
        q = s["q"]
        ctx.rope_append_device(s["handle"], case["tokens"], s["k"].data_ptr(), s["v"].data_ptr(),
                               rope=s["rope"], d_positions=s["positions"].data_ptr(),
                               d_q=q.data_ptr(), heads=case["heads"], q_token_stride=q.stride(1),
                               q_head_stride=q.stride(2), d_q_out=s["out"].data_ptr())
        return {"q": s["out"], "keys": s["cache"]["keys"], "values": s["cache"]["values"]}
    if kind == "attn":
        weights = s["weights"] if case["weights"] else None
        ctx.paged_attention_device(
            s["handle"], case["heads"], case["tokens"], s["scale"], s["q"].data_ptr(),
            s["out"].data_ptr(), s["scratch"].data_ptr(), s["scratch"].numel(),
            window=case["window"], d_counts=None if s["counts"] is None else s["counts"].data_ptr(),
            d_weights=None if weights is None else weights.data_ptr(),
            weights_stride=0 if weights is None else weights.shape[2])
        return s["out"] if weights is None else {"out": s["out"], "weights": weights}
    if kind == "evict":
        ctx.kv_evict_device(s["handle"], s["weights"].data_ptr(), s["weights"].shape[2],
                            case["keep"], case["sinks"], case["recent"], s["to_handle"],
                            s["to_weights"].data_ptr(), s["to_weights"].shape[2],
                            s["kept"].data_ptr())
        return _evicted(s)
    if kind == "softmax":
        ctx.softmax_device(s["x"].data_ptr(), case["rows"], case["cols"], case["temperature"],
                           s["out"].data_ptr())
        return s["out"]
    ctx.verify_draft_device(
        s["target"].data_ptr(), None if s["draft"] is None else s["draft"].data_ptr(),
        s["tokens"].data_ptr(), s["uniform"].data_ptr(), case["sequences"], case["drafts"],
        case["vocab"], s["accepted"].data_ptr(), s["out"].data_ptr(),
        d_counts=None if s["counts"] is None else s["counts"].data_ptr())
    return {"accepted": s["accepted"], "tokens": s["out"]}


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "softmax":
        n = case["rows"] * case["cols"]
        return {"bytes": 8 * n, "flops": 4.0 * n}
    if kind == "verify":  # one row of each, where the drafts end
        n = case["sequences"] * case["vocab"]
        return {"bytes": n * (4 if case["certain"] else 8), "flops": 3.0 * n}
    size, d, b = TYPES[case["type"]][1], case["head_dim"], case["sequences"]
    if kind == "rope":
        t = b * case["tokens"]
        rows = 4 * (2 * case["heads"] + 2 * case["kv_heads"]) + 2 * size * case["kv_heads"]
        return {"bytes": t * rows * d,
                "flops": 3.0 * t * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    if kind == "evict":
        left = sum(min(n, case["keep"]) for n in _lengths(case))
        return {"bytes": case["kv_heads"] * (4 * d * size * left + 8 * left + 4 * sum(_lengths(case))),
                "flops": 1.0 * case["kv_heads"] * sum(_lengths(case))}
    counts = _counts(case, case["tokens"])
    slots = pairs = 0
    for n, c in zip(_lengths(case), counts):
        seen = [min(n + t + 1, case["window"] or n + t + 1) for t in range(c)]
        pairs += sum(seen)
        slots += min(n + c, (case["window"] or n + c) + c - 1) if c else 0
    nbytes = slots * case["kv_heads"] * 2 * d * size + 8 * sum(counts) * case["heads"] * d
    return {"bytes": nbytes + (8 * slots * case["kv_heads"] if case["weights"] else 0),
            "flops": 4.0 * pairs * case["heads"] * d}


# ---- the same in 64 bits -----------------------------------------------------------

def _exact_rope(case, seed):
    q, k, v, positions, lengths = _rope_inputs(case, seed)
    cache = _cache(case, case["capacity"], lengths, seed, 10)
    inv, magnitude = _inverse_frequencies(case)
    angle = positions.double()[:, :, None, None] * torch.from_numpy(inv).cuda()
    turn = magnitude * torch.exp(1j * angle)
    n, d = case["rotary"], case["head_dim"]

    def rotated(x):
        y = x[..., :d].double().clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * turn
            y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :n].reshape(y.shape[:-1] + (n // 2, 2))) * turn
            y[..., :n] = torch.view_as_real(z).flatten(-2)
        return y

    keys, values = cache["keys"].double(), cache["values"].double()
    new = rotated(k)
    for i, length in enumerate(lengths):
        slot = torch.arange(length, length + case["tokens"], device="cuda")
        page = cache["table"][i].long()[slot // case["page"]]
        keys[page, :, slot % case["page"]] = new[i]
        values[page, :, slot % case["page"]] = v[i].double()
    return {"q": rotated(q), "keys": keys, "values": values}


def _exact_attn(case, seed):
    s = prepare(case, seed)
    c, d = s["cache"], case["head_dim"]
    g = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["weights"] else None
    counts = _counts(case, case["tokens"])
    for i, length in enumerate(_lengths(case)):
        pages = c["table"][i].long()[:-(-(length + case["tokens"]) // case["page"])]
        for h in range(case["kv_heads"]):
            k = c["keys"][pages, h].reshape(-1, d).double()
            v = c["values"][pages, h].reshape(-1, d).double()
            for t in range(counts[i]):
                end = length + t + 1
                begin = max(0, end - case["window"]) if case["window"] else 0
                q = s["q"][i, t, h * g:(h + 1) * g].double()
                p = torch.softmax(q @ k[begin:end].t().contiguous() * d ** -0.5, 1)
                out[i, t, h * g:(h + 1) * g] = p @ v[begin:end]
                if weights is not None:
                    weights[i, h, begin:end] += p.sum(0)
    return out if weights is None else {"out": out, "weights": weights}


def _exact_evict(case, seed):
    s = prepare(case, seed)
    c, to = s["cache"], s["to"]
    keys, values, kept = to["keys"].double(), to["values"].double(), torch.full_like(s["kept"], -1)
    weights = s["to_weights"].double()
    lengths = _lengths(case)
    for i, n in enumerate(lengths):
        left = min(n, case["keep"])
        at = torch.arange(left, device="cuda")
        page = to["table"][i].long()[at // case["page"]]
        for h in range(case["kv_heads"]):
            w = s["weights"][i, h, :n].double()
            rank = w.clone()
            rank[:case["sinks"]] = math.inf
            rank[max(0, n - case["recent"]):] = math.inf
            best = torch.sort(-rank, stable=True).indices[:left].sort().values
            source = c["table"][i].long()[best // case["page"]]
            keys[page, h, at % case["page"]] = c["keys"][source, h, best % case["page"]].double()
            values[page, h, at % case["page"]] = c["values"][source, h, best % case["page"]].double()
            weights[i, h, :left] = w[best]
            kept[i, h, :left] = best.to(torch.int32)
    return {"keys": keys, "values": values, "weights": weights, "kept": kept,
            "lengths": _ints([min(n, case["keep"]) for n in lengths])}


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None  # whole numbers
    if kind == "softmax":
        x = _logits(case["rows"], case["cols"], seed, 1).double() / case["temperature"]
        return torch.softmax(x, 1)
    return {"rope": _exact_rope, "attn": _exact_attn, "evict": _exact_evict}[kind](case, seed)
