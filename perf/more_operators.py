"""Performance cases of the mixers of a hybrid decoder layer on one MI355X.

Between the projections of such a layer a program runs, in an attention layer,
the norms of the query and key heads, their rotation by positions of one or
several axes and the append to the paged cache (one call), and, in a recurrent
layer, the short causal convolution over the projected channels and the scan
that keeps a matrix of state a head: the gated delta rule, or the selective
state space form without its correction.

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
RULES = ("delta", "selective")
ORDERS = ("grouped", "tiled")
AXIS_ORDERS = ("blocks", "turns")

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
        # one token of an attention layer: q lies beside its output gate, a quarter of a head turns
        {"name": "append_token", "kind": "append", "sequences": 1, "tokens": 1, "heads": 24,
         "kv_heads": 4, "head_dim": 256, "rotary": 64, "layout": "half", "sections": "32",
         "order": "blocks", "theta": 1e7, "plus_one": True, "gated": True, "type": "bf16",
         "page": 16, "capacity": 4096},
        # prompts with images in them: time, height and width take turns over a head's pairs
        {"name": "append_prompt", "kind": "append", "sequences": 4, "tokens": 2043, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rotary": 128, "layout": "half", "sections": "24,20,20",
         "order": "turns", "theta": 1e6, "plus_one": False, "gated": False, "type": "f16",
         "page": 64, "capacity": 4096},
        # query heads of a small picture's patches, row and column each half of the pairs
        {"name": "rows_patches", "kind": "rows", "tokens": 257, "heads": 16, "head_dim": 80,
         "rotary": 80, "layout": "half", "sections": "20,20", "order": "blocks", "theta": 1e4,
         "plus_one": False},
        # those of a video: pairs side by side, three axes
        {"name": "rows_video", "kind": "rows", "tokens": 30011, "heads": 16, "head_dim": 128,
         "rotary": 96, "layout": "interleaved", "sections": "16,16,16", "order": "blocks",
         "theta": 1e4, "plus_one": True},
        # one token of a recurrent layer: q, k and v channels behind one another
        {"name": "conv_token", "kind": "conv", "sequences": 1, "tokens": 1, "channels": 10240,
         "width": 4, "bias": False, "silu": True, "ragged": False, "fresh": False},
        # chunks of prompts of different lengths
        {"name": "conv_prompts", "kind": "conv", "sequences": 4, "tokens": 2043, "channels": 10240,
         "width": 4, "bias": True, "silu": True, "ragged": True, "fresh": False},
        # the next token of one conversation
        {"name": "scan_token", "kind": "scan", "rule": "delta", "sequences": 1, "tokens": 1,
         "key_heads": 16, "value_heads": 48, "key_dim": 128, "value_dim": 128, "order": "grouped",
         "skip": False, "ragged": False, "fresh": False, "keep": "both"},
        # the next tokens of a batch: the states' bytes are all of it
        {"name": "scan_batch", "kind": "scan", "rule": "delta", "sequences": 48, "tokens": 1,
         "key_heads": 16, "value_heads": 48, "key_dim": 128, "value_dim": 128, "order": "tiled",
         "skip": False, "ragged": False, "fresh": False, "keep": "both"},
        # drafted tokens of a few sequences; the states stay as they are until some are accepted
        {"name": "scan_verify", "kind": "scan", "rule": "delta", "sequences": 4, "tokens": 8,
         "key_heads": 16, "value_heads": 48, "key_dim": 128, "value_dim": 128, "order": "grouped",
         "skip": False, "ragged": True, "fresh": False, "keep": "out"},
        # one long prompt from its first token on
        {"name": "scan_prompt", "kind": "scan", "rule": "delta", "sequences": 1, "tokens": 4093,
         "key_heads": 16, "value_heads": 48, "key_dim": 128, "value_dim": 128, "order": "grouped",
         "skip": False, "ragged": False, "fresh": True, "keep": "both"},
        # later chunks of several prompts of different lengths
        {"name": "scan_prompts", "kind": "scan", "rule": "delta", "sequences": 8, "tokens": 2039,
         "key_heads": 16, "value_heads": 48, "key_dim": 128, "value_dim": 128, "order": "grouped",
         "skip": False, "ragged": True, "fresh": False, "keep": "both"},
        # the form without the correction, keys shared by many narrow heads, its input added
        {"name": "scan_selective", "kind": "scan", "rule": "selective", "sequences": 2,
         "tokens": 3001, "key_heads": 8, "value_heads": 64, "key_dim": 128, "value_dim": 64,
         "order": "grouped", "skip": True, "ragged": False, "fresh": False, "keep": "both"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _some_sections(rng, pairs, order):
    """The pairs of each axis: one axis, or two or three of them."""
    axes = rng.choice([1, 1, 2, 3])
    if axes == 1 or pairs < 6:
        return str(pairs)
    if order == "turns":
        rest = [(pairs - 1) // axes] * (axes - 1)
    else:
        rest = [rng.randint(1, pairs // axes) for _ in range(axes - 1)]
    return ",".join(str(n) for n in [pairs - sum(rest)] + rest)


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def draw(rng):
    kind = rng.choice(["append", "rows", "conv", "scan", "scan", "scan"])
    if kind in ("append", "rows"):
        heads, kv_heads, head_dim = rng.choice([(24, 4, 256), (32, 8, 128), (16, 16, 64),
                                                (32, 4, 128), (10, 2, 96), (8, 1, 192),
                                                (28, 4, 128), (40, 8, 80), (12, 12, 72)])
        rotary = rng.choice([head_dim, head_dim // 2, head_dim // 4])
        order = rng.choice(AXIS_ORDERS)
        shape = {"heads": heads, "head_dim": head_dim, "rotary": rotary,
                 "layout": rng.choice(["half", "interleaved"]),
                 "sections": _some_sections(rng, rotary // 2, order), "order": order,
                 "theta": rng.choice([1e4, 1e6, 1e7]), "plus_one": rng.random() < 0.5}
        if kind == "rows":
            return {"kind": kind, "tokens": _log(rng, 1, 60_000_000 // (heads * head_dim)), **shape}
        sequences = _log(rng, 1, 32)
        tokens = _log(rng, 1, 8000 // sequences)
        return {"kind": kind, "sequences": sequences, "tokens": tokens, "kv_heads": kv_heads, **shape,
                "gated": rng.random() < 0.3, "type": rng.choice(["f32", "f16", "bf16"]),
                "page": rng.choice([8, 16, 24, 32, 64, 128]),
                "capacity": tokens + _log(rng, 1, 2000)}
    if kind == "conv":
        channels = rng.choice([10240, 8192, 4352, 1537, 999])
        sequences = _log(rng, 1, 64)
        return {"kind": kind, "sequences": sequences, "tokens": _log(rng, 1, 8000 // sequences),
                "channels": channels, "width": rng.choice([2, 3, 4, 4, 4, 5, 8]),
                "bias": rng.random() < 0.5, "silu": rng.random() < 0.8,
                "ragged": rng.random() < 0.4, "fresh": rng.random() < 0.3}
    rule = rng.choice(["delta", "delta", "selective"])
    if rule == "delta":
        kh, vh, dk, dv = rng.choice([(16, 48, 128, 128), (16, 32, 128, 128), (8, 8, 64, 64),
                                     (6, 12, 96, 160), (4, 4, 192, 256), (5, 10, 40, 72)])
    else:
        kh, vh, dk, dv = rng.choice([(8, 64, 128, 64), (1, 24, 128, 64), (8, 80, 64, 64),
                                     (2, 32, 16, 80)])
    sequences = _log(rng, 1, 64)
    state = vh * dk * dv
    most = min(4000, 7500 * 786432 // max(state, 786432) // sequences)
    tokens = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 17, max(18, most)),
                         _log(rng, 17, max(18, most))])
    return {"kind": kind, "rule": rule, "sequences": sequences, "tokens": tokens, "key_heads": kh,
            "value_heads": vh, "key_dim": dk, "value_dim": dv, "order": rng.choice(ORDERS),
            "skip": rule == "selective" and rng.random() < 0.5,
            "ragged": tokens > 1 and rng.random() < 0.4, "fresh": rng.random() < 0.3,
            "keep": rng.choice(["both", "both", "out", "state"]) if tokens <= 16 else "both"}


# ---- inputs ------------------------------------------------------------------

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFFFFFF)


def _normal(shape, seed, salt, scale=1.0):
    return torch.randn(shape, generator=_generator(seed, salt), device="cuda") * scale


def _uniform(shape, seed, salt, lo, hi):
    return torch.rand(shape, generator=_generator(seed, salt), device="cuda") * (hi - lo) + lo


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _counts(case):
    """Each sequence's tokens: all of them, or a ragged number."""
    n, most = case["sequences"], case["tokens"]
    return [most if not case.get("ragged") or i % 3 == 0 else (i * 5 + 1) * most // (5 * n + 1)
            for i in range(n)]


def _axis_of_pairs(case):
    """The axis that each pair turns by."""
    sections = _sections(case)
    pairs, axes = case["rotary"] // 2, len(sections)
    if case["order"] == "blocks":
        return [a for a in range(axes) for _ in range(sections[a])]
    return [i % axes if i < axes * sections[i % axes] else 0 for i in range(pairs)]


def _inverse_frequencies(case):
    """Radians a position of each pair, in 64 bits: one ladder over the pairs, or for pictures, whose
    rows have no text among them, one for each block of pairs."""
    pairs = case["rotary"] // 2
    if case["kind"] == "rows" and case["order"] == "blocks":
        return np.concatenate([case["theta"] ** (-np.arange(n, dtype=np.float64) / n)
                               for n in _sections(case)])
    return case["theta"] ** (-np.arange(pairs, dtype=np.float64) / pairs)


def _frequencies(case):
    """The pairs' turns a position, as 64-bit fractions of a turn."""
    turns = _inverse_frequencies(case).astype(np.longdouble) / (2 * np.longdouble(np.pi))
    table = np.rint(turns * np.longdouble(2.0) ** 64).astype(np.uint64)
    return torch.from_numpy(table.view(np.int64)).cuda()


def _positions(case, rows, seed):
    """[axes][rows]: a row's place in time, and in each further axis of a picture."""
    axes = len(_sections(case))
    n = case["tokens"]
    first = torch.randint(0, 100_000, (rows // n, 1), generator=_generator(seed, 4), device="cuda")
    step = torch.arange(n, device="cuda")
    out = [(first + (step if axes == 1 else step // 64)).reshape(-1)]
    for a in range(1, axes):
        out.append((first * (case["kind"] == "append") + (step * (7 if a == 1 else 1)) % 64).reshape(-1))
    return torch.stack(out).to(torch.int32)


def _norm_inputs(case, seed):
    d = case["head_dim"]
    weight = _normal((2, d), seed, 6, 0.2) + (0.0 if case["plus_one"] else 1.0)
    if case["kind"] == "rows":
        return _normal((case["tokens"], case["heads"], d), seed, 1, 3.0), weight
    b, t = case["sequences"], case["tokens"]
    q = _normal((b, t, case["heads"], (2 if case["gated"] else 1) * d), seed, 1, 3.0)
    k = _normal((b, t, case["kv_heads"], d), seed, 2, 5.0)
    v = _normal((b, t, case["kv_heads"], d), seed, 3)
    return q, k, v, weight


def _cache(case, seed):
    max_pages = -(-case["capacity"] // case["page"])
    n = case["sequences"]
    order = torch.randperm(n * max_pages, generator=_generator(seed, 10), device="cuda")
    lengths = [(case["capacity"] - case["tokens"]) * (i + 1) // n for i in range(n)]
    shape = (n * max_pages, case["kv_heads"], case["page"], case["head_dim"])
    kind = TYPES[case["type"]][0]
    keys = torch.randn(shape, generator=_generator(seed, 11), device="cuda").to(kind)
    values = torch.randn(shape, generator=_generator(seed, 12), device="cuda").to(kind)
    return {"table": order.view(n, max_pages).to(torch.int32), "lengths": _ints(lengths),
            "keys": keys, "values": values}


def _conv_inputs(case, seed):
    b, t, c, w = case["sequences"], case["tokens"], case["channels"], case["width"]
    return {"x": _normal((b, t, c), seed, 1), "weight": _normal((c, w), seed, 2, w ** -0.5),
            "bias": _normal((c,), seed, 3, 0.1) if case["bias"] else None,
            "state": None if case["fresh"] else _normal((b, w - 1, c), seed, 4)}


def _scan_inputs(case, seed):
    b, t = case["sequences"], case["tokens"]
    kh, vh, dk, dv = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
    # what the convolution and its activation leave: q, k and v of a token behind one another
    x = _normal((b, t, 2 * kh * dk + vh * dv), seed, 1)
    step = torch.exp(_uniform((vh,), seed, 5, math.log(1e-3), math.log(0.1)))
    return {"qkv": x * torch.sigmoid(x), "gate": _normal((b, t, vh), seed, 2),
            "beta": _normal((b, t, vh), seed, 3) if case["rule"] == "delta" else None,
            "decay": -_uniform((vh,), seed, 4, 1.0, 16.0),
            "bias": step + torch.log(-torch.expm1(-step)),
            "skip": _normal((vh,), seed, 6, 0.3) + 1.0 if case["skip"] else None,
            "state": None if case["fresh"] else _normal((b, vh, dk, dv), seed, 7, 0.2)}


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if kind in ("append", "rows"):
        inputs = _norm_inputs(case, seed)
        if kind == "append":
            s["q"], s["k"], s["v"], s["weight"] = inputs
            s["cache"] = _cache(case, seed)
            rows = case["sequences"] * case["tokens"]
        else:
            s["q"], s["weight"] = inputs
            rows = case["tokens"]
        s["positions"] = _positions(case, rows, seed)
        s["table"] = _frequencies(case)
        s["axis"] = torch.tensor(_axis_of_pairs(case), dtype=torch.uint8, device="cuda")
        s["out"] = torch.empty(s["q"].shape[:-1] + (case["head_dim"],), device="cuda")
    else:
        s.update(_conv_inputs(case, seed) if kind == "conv" else _scan_inputs(case, seed))
        s["counts"] = _ints(_counts(case)) if case["ragged"] else None
        # (rows behind a sequence's tokens stay as they are)
        if kind == "conv":
            s["out"] = torch.zeros_like(s["x"])
            s["new_state"] = s["state"] if s["state"] is not None else torch.empty(
                (case["sequences"], case["width"] - 1, case["channels"]), device="cuda")
        else:
            b, t, vh = case["sequences"], case["tokens"], case["value_heads"]
            s["out"] = torch.zeros((b, t, vh, case["value_dim"]), device="cuda")
            s["new_state"] = s["state"] if s["state"] is not None else torch.empty(
                (b, vh, case["key_dim"], case["value_dim"]), device="cuda")
    if own:  # what a program makes once and keeps: its context and its descriptions
        si_hip = _package()
        s["ctx"] = _context()
        if kind in ("append", "rows"):
            s["norm"] = si_hip.HeadNorm(eps=1e-6, plus_one=int(case["plus_one"]),
                                        d_q_weight=s["weight"][0].data_ptr(),
                                        d_k_weight=s["weight"][1].data_ptr())
            s["rope"] = si_hip.Rope(layout=("half", "interleaved").index(case["layout"]),
                                    rotary_dim=case["rotary"], magnitude=1.0,
                                    d_frequencies=s["table"].data_ptr())
            s["axes"] = None
            if len(_sections(case)) > 1:
                s["axes"] = si_hip.RopeAxes(axes=len(_sections(case)), d_axis=s["axis"].data_ptr())
        if kind == "append":
            c = s["cache"]
            s["handle"] = si_hip.KvCache(
                ggml_type=TYPES[case["type"]][2], kv_heads=case["kv_heads"],
                head_dim=case["head_dim"], page_tokens=case["page"], pages=c["keys"].shape[0],
                sequences=case["sequences"], max_pages=c["table"].shape[1],
                d_keys=c["keys"].data_ptr(), d_values=c["values"].data_ptr(),
                d_page_table=c["table"].data_ptr(), d_lengths=c["lengths"].data_ptr())
        if kind == "scan":
            s["scan"] = si_hip.StateScan(
                rule=RULES.index(case["rule"]), head_order=ORDERS.index(case["order"]),
                key_heads=case["key_heads"], value_heads=case["value_heads"],
                key_dim=case["key_dim"], value_dim=case["value_dim"], scale=_scale(case), eps=1e-6,
                d_decay=s["decay"].data_ptr(), d_bias=s["bias"].data_ptr(),
                d_skip=None if s["skip"] is None else s["skip"].data_ptr())
    return s


def _scale(case):
    return case["key_dim"] ** -0.5 if case["rule"] == "delta" else 1.0


# ---- the operators in plain form -----------------------------------------------

def _normed(s, x, which):
    case = s["case"]
    w = s["weight"][which] + (1.0 if case["plus_one"] else 0.0)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _rotate(s, x):
    """x [rows][heads][d] with its first values turned by the row's positions."""
    case = s["case"]
    # the fraction of a turn, exact in wrapping 64-bit integers, then 32 bits
    position = s["positions"].long()[s["axis"].long()].t()
    angle = (position * s["table"]).float()[:, None] * (2.0 ** -64 * 2 * math.pi)
    cos, sin = torch.cos(angle), torch.sin(angle)
    n = case["rotary"] // 2
    if case["layout"] == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rows(s):
    return _rotate(s, _normed(s, s["q"], 0))


def _plain_append(s):
    case, c = s["case"], s["cache"]
    d = case["head_dim"]
    q = _rotate(s, _normed(s, s["q"][..., :d], 0).flatten(0, 1)).view(s["out"].shape)
    k = _rotate(s, _normed(s, s["k"], 1).flatten(0, 1)).view(s["k"].shape)
    slots = c["lengths"].long()[:, None] + torch.arange(case["tokens"], device="cuda")
    page, row = c["table"].long().gather(1, slots // case["page"]), slots % case["page"]
    c["keys"][page, :, row] = k.to(c["keys"].dtype)
    c["values"][page, :, row] = s["v"].to(c["values"].dtype)
    return {"q": q, "keys": c["keys"], "values": c["values"]}


def _there(s):
    """[sequences][tokens]: the rows that are a sequence's."""
    case = s["case"]
    counts = _ints([case["tokens"]] * case["sequences"]) if s["counts"] is None else s["counts"]
    return torch.arange(case["tokens"], device="cuda") < counts[:, None], counts.long()


def _plain_conv(s):
    case = s["case"]
    width = case["width"]
    there, counts = _there(s)
    old = s["state"]
    if old is None:
        old = torch.zeros((case["sequences"], width - 1, case["channels"]), device="cuda")
    rows = torch.cat([old, s["x"]], 1)
    y = sum(rows[:, j:j + case["tokens"]] * s["weight"][:, j] for j in range(width))
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["silu"]:
        y = y / (1.0 + torch.exp(-y))
    last = counts[:, None] + torch.arange(width - 1, device="cuda")
    state = rows.gather(1, last[:, :, None].expand(-1, -1, case["channels"]))
    s["new_state"].copy_(state)
    return {"out": torch.where(there[:, :, None], y, torch.zeros_like(y)), "state": s["new_state"]}


def _heads_of(case, x):
    """[.., key_heads, d] as the value heads see it."""
    group = case["value_heads"] // case["key_heads"]
    if case["order"] == "grouped":
        return x.repeat_interleave(group, -2)
    return torch.cat([x] * group, -2)


def _split(case, qkv):
    b, t = qkv.shape[:2]
    n = case["key_heads"] * case["key_dim"]
    shape = (b, t, case["key_heads"], case["key_dim"])
    return (qkv[..., :n].view(shape), qkv[..., n:2 * n].view(shape),
            qkv[..., 2 * n:].view(b, t, case["value_heads"], case["value_dim"]))


def _plain_scan(s):
    case = s["case"]
    delta = case["rule"] == "delta"
    there, _ = _there(s)
    q, k, v = _split(case, s["qkv"])
    if delta:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q, k = _heads_of(case, q * _scale(case)), _heads_of(case, k)
    x = s["gate"] + s["bias"]
    step = x.clamp(min=0.0) + torch.log1p(torch.exp(-x.abs()))
    keep = torch.exp(s["decay"] * step)
    write = 1.0 / (1.0 + torch.exp(-s["beta"])) if delta else step
    # a row that is none of the sequence's leaves its state as it is
    keep = torch.where(there[..., None], keep, torch.ones_like(keep))
    write = torch.where(there[..., None], write, torch.zeros_like(write))
    state = s["new_state"] if case["keep"] != "out" else torch.empty_like(s["new_state"])
    if s["state"] is None:
        state.zero_()
    elif case["keep"] == "out":
        state.copy_(s["state"])
    out = torch.empty_like(s["out"])
    for t in range(case["tokens"]):
        state *= keep[:, t, :, None, None]
        u = v[:, t]
        if delta:
            u = u - (state * k[:, t, :, :, None]).sum(-2)
        state += k[:, t, :, :, None] * (write[:, t, :, None] * u)[:, :, None]
        out[:, t] = (state * q[:, t, :, :, None]).sum(-2)
    if s["skip"] is not None:
        out = out + s["skip"][:, None] * v
    out = torch.where(there[:, :, None, None], out, torch.zeros_like(out))
    return _scanned(case, out, state)


def _scanned(case, out, state):
    if case["keep"] == "both":
        return {"out": out, "state": state}
    return out if case["keep"] == "out" else state


# ---- one pass ------------------------------------------------------------------

def run(state):
    s = state
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"append": _plain_append, "rows": _plain_rows, "conv": _plain_conv,
                "scan": _plain_scan}[kind](s)
    ctx = s["ctx"]
    at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    if kind == "rows":
        ctx.norm_rope_device(at(s["q"]), case["tokens"], case["heads"], case["head_dim"],
                             at(s["out"]), norm=s["norm"], rope=s["rope"], axes=s["axes"],
                             d_positions=at(s["positions"]))
        return s["out"]
    if kind == "append":
        q = s["q"]
        ctx.norm_rope_append_device(
            s["handle"], case["tokens"], at(s["k"]), at(s["v"]), norm=s["norm"], rope=s["rope"],
            axes=s["axes"], d_positions=at(s["positions"]), d_q=at(q), heads=case["heads"],
            q_token_stride=q.stride(1), q_head_stride=q.stride(2), d_q_out=at(s["out"]))
        return {"q": s["out"], "keys": s["cache"]["keys"], "values": s["cache"]["values"]}
    if kind == "conv":
        si_hip = _package()
        ctx.causal_conv_device(
            at(s["x"]), at(s["weight"]), case["sequences"], case["tokens"], case["channels"],
            case["width"], d_y=at(s["out"]), d_bias=at(s["bias"]),
            activation=si_hip.CONV_SILU if case["silu"] else si_hip.CONV_NONE,
            d_state=at(s["state"]), d_state_out=at(s["new_state"]), d_counts=at(s["counts"]))
        return {"out": s["out"], "state": s["new_state"]}
    x, n = s["qkv"], case["key_heads"] * case["key_dim"]
    ctx.state_scan_device(
        s["scan"], case["sequences"], case["tokens"], at(x), at(x) + 4 * n, at(x) + 8 * n,
        at(s["gate"]), d_beta=at(s["beta"]), d_state=at(s["state"]),
        d_state_out=None if case["keep"] == "out" else at(s["new_state"]),
        d_out=None if case["keep"] == "state" else at(s["out"]), d_counts=at(s["counts"]),
        q_token_stride=x.stride(1), k_token_stride=x.stride(1), v_token_stride=x.stride(1))
    return _scanned(case, s["out"], s["new_state"])


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("append", "rows"):
        d = case["head_dim"]
        heads, b = 2 * case["heads"], case["tokens"]
        rows = 4 * heads
        turned = case["heads"]
        if kind == "append":
            size = TYPES[case["type"]][1]
            b *= case["sequences"]
            rows += (8 + 2 * size) * case["kv_heads"]
            turned += case["kv_heads"]
        return {"bytes": b * (rows * d + 4 * len(_sections(case))),
                "flops": b * turned * (4.0 * d + 3.0 * case["rotary"])}
    counts = _counts(case)
    total = sum(counts)
    if kind == "conv":
        c, w = case["channels"], case["width"]
        states = case["sequences"] * (1 if case["fresh"] else 2) * (w - 1)
        return {"bytes": 4 * c * (2 * total + states + w), "flops": 2.0 * total * c * w}
    kh, vh, dk, dv = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
    delta = case["rule"] == "delta"
    outs, states = case["keep"] != "state", (not case["fresh"]) + (case["keep"] != "out")
    row = (2 if outs else 1) * kh * dk + (2 if outs else 1) * vh * dv + (2 if delta else 1) * vh
    products = 2 * (outs + 1 + delta)
    return {"bytes": 4 * (total * row + case["sequences"] * states * vh * dk * dv),
            "flops": 1.0 * total * vh * dk * dv * products}


# ---- the same in 64 bits -----------------------------------------------------------

def _exact_norm(case, seed):
    inputs = _norm_inputs(case, seed)
    rows = case["tokens"] * case.get("sequences", 1)
    positions = _positions(case, rows, seed).double()
    inv = torch.from_numpy(_inverse_frequencies(case)).cuda()
    angle = torch.stack([positions[a] * inv[i] for i, a in enumerate(_axis_of_pairs(case))], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    n, d = case["rotary"], case["head_dim"]

    def turned(x, weight):
        w = weight.double() + (1 if case["plus_one"] else 0)
        y = x.double().reshape(rows, -1, x.shape[-1])[..., :d]
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        if case["layout"] == "half":
            z = torch.complex(y[..., :n // 2], y[..., n // 2:n].clone()) * turn
            y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :n].reshape(y.shape[:-1] + (n // 2, 2))) * turn
            y[..., :n] = torch.view_as_real(z).flatten(-2)
        return y.view(x.shape[:-1] + (d,))

    if case["kind"] == "rows":
        return turned(inputs[0], inputs[1][0])
    q, k, v, weight = inputs
    cache = _cache(case, seed)
    keys, values = cache["keys"].double(), cache["values"].double()
    new = turned(k, weight[1])
    for i, length in enumerate(cache["lengths"].tolist()):
        slot = torch.arange(length, length + case["tokens"], device="cuda")
        page = cache["table"][i].long()[slot // case["page"]]
        keys[page, :, slot % case["page"]] = new[i]
        values[page, :, slot % case["page"]] = v[i].double()
    return {"q": turned(q, weight[0]), "keys": keys, "values": values}


def _exact_conv(case, seed):
    i = _conv_inputs(case, seed)
    width, channels = case["width"], case["channels"]
    out = torch.zeros(i["x"].shape, dtype=torch.float64, device="cuda")
    states = []
    for b, count in enumerate(_counts(case)):
        old = torch.zeros((width - 1, channels), dtype=torch.float64, device="cuda")
        if i["state"] is not None:
            old = i["state"][b].double()
        rows = torch.cat([old, i["x"][b, :count].double()])
        states.append(rows[count:])
        if count == 0:
            continue
        y = (rows.unfold(0, width, 1) * i["weight"].double()).sum(-1)
        if i["bias"] is not None:
            y = y + i["bias"].double()
        out[b, :count] = y * torch.sigmoid(y) if case["silu"] else y
    return {"out": out, "state": torch.stack(states)}


def _exact_scan(case, seed):
    i = _scan_inputs(case, seed)
    vh, dk, dv = case["value_heads"], case["key_dim"], case["value_dim"]
    group = vh // case["key_heads"]
    heads = torch.arange(vh, device="cuda")
    heads = heads // group if case["order"] == "grouped" else heads % case["key_heads"]
    delta = case["rule"] == "delta"
    q, k, v = (x.double() for x in _split(case, i["qkv"]))
    if delta:
        q, k = (x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q, k = q[:, :, heads] * _scale(case), k[:, :, heads]
    step = torch.nn.functional.softplus(i["gate"].double() + i["bias"].double(), threshold=60.0)
    log_keep = i["decay"].double() * step
    write = torch.sigmoid(i["beta"].double()) if delta else step
    out = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    states = torch.zeros((case["sequences"], vh, dv, dk), dtype=torch.float64, device="cuda")
    if i["state"] is not None:
        states += i["state"].double().transpose(2, 3)
    counts = _counts(case)
    # sequences longest first, those that are through leave from the end
    order = sorted(range(case["sequences"]), key=lambda n: -counts[n])
    part = states[order]
    q, k, v, log_keep, write = (x[order] for x in (q, k, v, log_keep, write))
    made = torch.zeros_like(out)
    for t in range(case["tokens"]):
        n = sum(c > t for c in counts)
        if n == 0:
            break
        before = part[:n] * torch.exp(log_keep[:n, t])[:, :, None, None]
        add = v[:n, t]
        if delta:
            add = add - torch.matmul(before, k[:n, t, :, :, None])[..., 0]
        before += (add * write[:n, t, :, None])[..., None] * k[:n, t, :, None]
        made[:n, t] = torch.matmul(before, q[:n, t, :, :, None])[..., 0]
        if i["skip"] is not None:
            made[:n, t] += i["skip"].double()[:, None] * v[:n, t]
        part[:n] = before
    out[order], states[order] = made, part
    return _scanned(case, out, states.transpose(2, 3).contiguous())


def exact(case, seed):
    if case["kind"] in ("append", "rows"):
        return _exact_norm(case, seed)
    return (_exact_conv if case["kind"] == "conv" else _exact_scan)(case, seed)
