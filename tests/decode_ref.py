"""The decode-step operators (include/si_hip_decode.h) in 64 bits on the CPU,
and device arrays for their tests."""
from __future__ import annotations

import numpy as np

import si_hip

NONE = si_hip.TOKEN_NONE
TYPES = {"f32": (si_hip.GGML_TYPE_F32, np.float32), "f16": (si_hip.GGML_TYPE_F16, np.float16),
         "bf16": (si_hip.GGML_TYPE_BF16, np.uint16)}


def to_bf16(x) -> np.ndarray:
    """Nearest bf16 bits, ties to even; a NaN stays one."""
    x = np.ascontiguousarray(x, np.float32)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b) -> np.ndarray:
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def encode(x, kind) -> np.ndarray:
    return to_bf16(x) if kind == "bf16" else np.asarray(x, np.float32).astype(TYPES[kind][1])


def decode(b, kind) -> np.ndarray:
    return from_bf16(b) if kind == "bf16" else np.asarray(b).astype(np.float32)


class Device:
    """Arrays in device memory; `offset` moves one off its allocation's alignment."""

    def __init__(self, ctx):
        self.ctx, self.held = ctx, []

    def raw(self, nbytes: int) -> int:
        p = self.ctx.device_alloc(max(int(nbytes), 1))
        self.held.append(p)
        return p

    def put(self, a, offset: int = 0) -> int:
        a = np.ascontiguousarray(a)
        p = self.raw(a.nbytes + offset) + offset
        if a.nbytes:
            self.ctx.to_device(p, a)
        return p

    def get(self, p: int, like) -> np.ndarray:
        return self.ctx.from_device(p, like.shape, like.dtype)

    def free(self):
        for p in self.held:
            self.ctx.device_free(p)
        self.held = []


class Cache:
    """A paged cache whose pages lie in random order, host copy and device arrays."""

    def __init__(self, dev, rng, kind, sequences, kv_heads, head_dim, page, max_pages, lengths,
                 offset=0, spare=3, fill=1.0):
        self.kind, self.page, self.max_pages = kind, page, max_pages
        self.kv_heads, self.head_dim = kv_heads, head_dim
        pages = sequences * max_pages + spare
        shape = (pages, kv_heads, page, head_dim)
        self.keys = encode(rng.standard_normal(shape) * fill, kind)
        self.values = encode(rng.standard_normal(shape) * fill, kind)
        self.table = rng.permutation(pages)[:sequences * max_pages].astype(np.uint32).reshape(
            sequences, max_pages)
        self.lengths = np.asarray(lengths, np.uint32)
        self.dev, self.offset = dev, offset
        self.upload()

    def upload(self):
        d = self.dev
        self.d_keys, self.d_values = d.put(self.keys, self.offset), d.put(self.values, self.offset)
        self.d_table, self.d_lengths = d.put(self.table), d.put(self.lengths)
        self.handle = si_hip.KvCache(
            ggml_type=TYPES[self.kind][0], kv_heads=self.kv_heads, head_dim=self.head_dim,
            page_tokens=self.page, pages=self.keys.shape[0], sequences=len(self.lengths),
            max_pages=self.max_pages, d_keys=self.d_keys, d_values=self.d_values,
            d_page_table=self.d_table, d_lengths=self.d_lengths)

    @property
    def capacity(self):
        return self.max_pages * self.page

    def at(self, seq, slot):
        return int(self.table[seq, slot // self.page]), slot % self.page

    def rows(self, what, seq, head, slots) -> np.ndarray:
        """Rows of slots in f64: [len(slots)][head_dim]."""
        slots = np.asarray(slots, np.int64)
        a = getattr(self, what)[self.table[seq, slots // self.page], head, slots % self.page]
        return decode(a, self.kind).astype(np.float64)

    def device(self, what):
        return self.dev.get(getattr(self, "d_" + what), getattr(self, what))


# ---- rotary positions --------------------------------------------------------------

def inverse_frequencies(n, theta, scaling="none", factor=4.0, original=32768.0, fast=32.0, slow=1.0):
    i = np.arange(n // 2, dtype=np.float64)
    inv = theta ** (-2.0 * i / n)
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "yarn":
        dim = lambda t: n * np.log(original / (t * 2 * np.pi)) / (2 * np.log(theta))  # noqa: E731
        low, high = max(np.floor(dim(fast)), 0), min(np.ceil(dim(slow)), n - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * np.log(factor) + 1
    return inv, 1.0


def rotate(x, positions, inv, magnitude, layout):
    """x [rows][heads][dim] in f64, and what bounds each value's error (the
    magnitude of its pair)."""
    x = np.asarray(x, np.float64).copy()
    size = np.abs(x)
    h = len(inv)
    angle = np.asarray(positions, np.float64)[:, None, None] * inv
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    ia = np.arange(h) if layout == si_hip.ROPE_HALF else np.arange(0, 2 * h, 2)
    ib = ia + h if layout == si_hip.ROPE_HALF else ia + 1
    a, b = x[..., ia].copy(), x[..., ib].copy()
    x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = (np.abs(a) + np.abs(b)) * magnitude
    return x, size


# ---- attention -----------------------------------------------------------------------

def attention(cache, q, scale, window, counts, walk=4096):
    """out, its tolerance, weights [sequences][kv_heads][capacity] and theirs.

    The tolerance: an f32 score of d terms is off by about 16 units in the last
    place of sum |q k| (d <= 256 roundings, a random walk), which moves p by as
    much on both sides of its fraction; the sums over the slots add a walk of
    their own, 64 units for up to 4096 slots and with the root of `walk` slots above.
    """
    sums = 64 * max(1.0, walk / 4096) ** 0.5
    b, t, h, d = q.shape
    g = h // cache.kv_heads
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    w = np.zeros((b, cache.kv_heads, cache.capacity))
    wtol = np.zeros_like(w)
    for s in range(b):
        n = min(int(cache.lengths[s]), cache.capacity)
        for i in range(t if counts is None else min(int(counts[s]), t)):
            end = min(n + i + 1, cache.capacity)
            begin = max(0, n + i + 1 - window) if window else 0
            slots = np.arange(begin, end)
            slots = slots[cache.table[s, slots // cache.page] < cache.keys.shape[0]]
            if not len(slots):
                continue
            for kv in range(cache.kv_heads):
                k, v = cache.rows("keys", s, kv, slots), cache.rows("values", s, kv, slots)
                for j in range(kv * g, (kv + 1) * g):
                    x = q[s, i, j].astype(np.float64)
                    score = k @ x * scale
                    p = np.exp(score - score.max())
                    p /= p.sum()
                    out[s, i, j] = p @ v
                    big = float((np.abs(k) @ np.abs(x)).max()) * abs(scale)
                    rel = (2 * 16 * big + sums) * 2.0 ** -24
                    tol[s, i, j] = rel * (p @ np.abs(v)) + 1e-30
                    w[s, kv, slots] += p
                    wtol[s, kv, slots] += p * rel + 1e-30
    return out, tol, w, wtol


# ---- eviction ------------------------------------------------------------------------

def kept_slots(w, n, keep, sinks, recent):
    """The slots one head keeps of n."""
    if n <= keep:
        return np.arange(n)
    nan = np.isnan(w[:n])  # below -inf
    w = np.where(nan, -np.inf, w[:n].astype(np.float64))
    inside = np.arange(sinks, n - recent)
    order = sorted(inside, key=lambda i: (nan[i], -w[i], i))[:keep - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), np.asarray(order, int),
                                   np.arange(n - recent, n)]).astype(int))


# ---- verification --------------------------------------------------------------------

def fixed(x):
    x = np.asarray(x, np.float32).astype(np.float64)
    x = np.where(np.isnan(x), 0.0, np.clip(x, 0.0, 1.0))
    return [int(v) for v in np.floor(x * 2.0 ** 36)]


def verify(target, draft, tokens, counts, uniform, vocab):
    n, m = tokens.shape
    accepted = np.zeros(n, np.uint32)
    out = np.full((n, m + 1), NONE, np.uint32)
    for s in range(n):
        count = m if counts is None else min(int(counts[s]), m)
        i = 0
        while i < count:
            x = int(tokens[s, i])
            if x >= vocab:
                break
            q = np.float32(1.0) if draft is None else draft[s, i, x]
            if not np.float32(uniform[s, i] * q) < target[s, i, x]:
                break
            i += 1
        accepted[s] = i
        out[s, :i] = tokens[s, :i]
        p = target[s, i]
        rest = fixed(p)
        if i < count:
            if draft is not None:
                rest = fixed(p - draft[s, i])
            else:
                r = p.copy()
                if int(tokens[s, i]) < vocab:
                    r[int(tokens[s, i])] -= np.float32(1.0)
                rest = fixed(r)
        if sum(rest) == 0:
            rest = fixed(p)
        total = sum(rest)
        if total == 0:
            continue
        u = float(uniform[s, m])
        n24 = min(int(u * 2 ** 24), 2 ** 24 - 1) if u > 0 else 0
        threshold = (n24 * total) >> 24
        running = 0
        for v, r in enumerate(rest):
            running += r
            if running > threshold:
                out[s, i] = v
                break
    return accepted, out
