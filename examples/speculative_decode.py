"""Speculative decoding over a paged cache that evicts: the device side of a
decode step, captured once and replayed.

A one-layer decoder with random K-quant weights: embedding, norm, q / k / v,
rotary positions into the cache, attention that adds up each cached token's
weight, the output projection, the head, probabilities, and the verification of
tokens that an n-gram drafter proposes from what was generated so far.  When a
sequence has no room for the next step, every head keeps its heaviest tokens
(the first few and the latest ones anyway) on other pages of the same pool.

    python examples/speculative_decode.py --steps 100
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "memory-aware-inference_amd"))
import si_hip  # noqa: E402
from si_hip import GGML_TYPE_Q4_K, GGML_TYPE_Q6_K  # noqa: E402


def centred_blocks(rng, kind: int, blocks: int, deviation: float) -> np.ndarray:
    """K-quant blocks of evenly spread quants around zero, with the given deviation."""
    if kind == GGML_TYPE_Q4_K:  # d, dmin, 6-bit scales and minima (all 1), 4-bit quants
        d = np.float16(deviation / np.sqrt((16 ** 2 - 1) / 12))
        head = np.array([d, np.float16(7.5) * d], np.float16).tobytes() + b"\1" * 8 + b"\x11" * 4
        quants = rng.integers(0, 256, (blocks, 128), np.uint8)
        return np.concatenate([np.tile(np.frombuffer(head, np.uint8), (blocks, 1)), quants], 1).ravel()
    # Q6_K: 4 low and 2 high bits a quant, 8-bit scales (all 1), d
    tail = b"\1" * 16 + np.float16(deviation / np.sqrt((64 ** 2 - 1) / 12)).tobytes()
    quants = rng.integers(0, 256, (blocks, 192), np.uint8)
    return np.concatenate([quants, np.tile(np.frombuffer(tail, np.uint8), (blocks, 1))], 1).ravel()


class Drafter:
    """Proposes what followed the last occurrence of the latest token."""

    def propose(self, tokens: list[int], count: int) -> list[int]:
        for at in range(len(tokens) - 2, -1, -1):
            if tokens[at] == tokens[-1]:
                followed = tokens[at + 1:]
                return [followed[i % len(followed)] for i in range(count)]
        return [tokens[-1]] * count


class SpeculativeDecoder:
    def __init__(self, ctx, sequences=2, drafts=3, hidden=512, heads=8, kv_heads=2, head_dim=64,
                 vocab=1024, page_tokens=16, capacity=64, keep=40, sinks=4, recent=12,
                 temperature=0.15, cache_type=si_hip.GGML_TYPE_BF16, seed=1, use_graph=True):
        self.ctx, self.lib = ctx, si_hip.lib()
        self.sequences, self.drafts, self.vocab = sequences, drafts, vocab
        self.hidden, self.heads, self.head_dim, self.kv_heads = hidden, heads, head_dim, kv_heads
        self.keep, self.sinks, self.recent = keep, sinks, recent
        self.temperature, self.use_graph = temperature, use_graph
        self.tokens = drafts + 1  # rows a sequence brings to a step
        self.rows = sequences * self.tokens
        self.rng = np.random.default_rng(seed)
        self.buffers = []

        def weight(kind, rows):
            blocks = centred_blocks(self.rng, kind, rows * (hidden // 256), hidden ** -0.5)
            return ctx.upload_quant_weight_private(blocks, kind)

        self.embed = weight(GGML_TYPE_Q4_K, vocab)
        self.w_q = weight(GGML_TYPE_Q4_K, heads * head_dim)
        self.w_k = weight(GGML_TYPE_Q4_K, kv_heads * head_dim)
        self.w_v = weight(GGML_TYPE_Q4_K, kv_heads * head_dim)
        if heads * head_dim != hidden:
            raise ValueError("this example's output projection is square")
        self.w_o = weight(GGML_TYPE_Q4_K, hidden)
        self.head = weight(GGML_TYPE_Q6_K, vocab)
        self.norm = self.put(np.zeros(hidden, np.float32))  # (1 + w) norms

        table, magnitude = si_hip.rope_frequencies(head_dim, 1e6)
        self.rope = si_hip.Rope(layout=si_hip.ROPE_HALF, rotary_dim=head_dim, magnitude=magnitude,
                                d_frequencies=self.put(table))
        # one pool, two sets of pages a sequence: eviction moves from one to the other
        max_pages = -(-capacity // page_tokens)
        self.capacity = max_pages * page_tokens
        pages = 2 * sequences * max_pages
        size = 4 if cache_type == si_hip.GGML_TYPE_F32 else 2
        pool = pages * kv_heads * page_tokens * head_dim * size
        keys, values = self.raw(pool), self.raw(pool)
        order = self.rng.permutation(pages).astype(np.uint32).reshape(2, sequences, max_pages)
        self.caches, self.weights = [], []
        self.page_tables = order
        for which in range(2):
            self.caches.append(si_hip.KvCache(
                ggml_type=cache_type, kv_heads=kv_heads, head_dim=head_dim,
                page_tokens=page_tokens, pages=pages, sequences=sequences, max_pages=max_pages,
                d_keys=keys, d_values=values, d_page_table=self.put(order[which]),
                d_lengths=self.put(np.zeros(sequences, np.uint32))))
            self.weights.append(self.put(np.zeros((sequences, kv_heads, self.capacity), np.float32)))
        self.kept = self.raw(sequences * kv_heads * keep * 4)

        n, h = self.rows, hidden
        f32 = lambda *shape: self.raw(4 * int(np.prod(shape)))  # noqa: E731
        self.d_ids, self.d_positions = f32(n), f32(n)
        self.d_drafts, self.d_uniform = f32(sequences, drafts), f32(sequences, drafts + 1)
        self.d_x, self.d_h, self.d_attn, self.d_o = f32(n, h), f32(n, h), f32(n, h), f32(n, h)
        self.d_q, self.d_q_rot = f32(n, h), f32(n, h)
        self.d_k, self.d_v = f32(n, kv_heads * head_dim), f32(n, kv_heads * head_dim)
        self.d_logits, self.d_probs = f32(n, vocab), f32(n, vocab)
        self.d_accepted, self.d_next = f32(sequences), f32(sequences, drafts + 1)
        self.space_bytes = ctx.paged_attention_workspace(self.caches[0], heads, self.tokens, True)
        self.space = self.raw(self.space_bytes)

        self.now = 0  # the cache in use
        self.lengths = np.zeros(sequences, np.int64)  # tokens it holds
        self.text = [[int(t)] for t in self.rng.integers(0, vocab, sequences)]
        self.drafter = Drafter()
        self.graphs = [self._capture(which) for which in range(2)] if use_graph else None
        self.evictions = 0

    # ---- device memory
    def raw(self, nbytes: int) -> int:
        p = self.ctx.device_alloc(max(nbytes, 4))
        self.buffers.append(p)
        return p

    def put(self, a) -> int:
        p = self.raw(a.nbytes)
        self.ctx.to_device(p, np.ascontiguousarray(a))
        return p

    def close(self) -> None:
        self.ctx.synchronize()
        for g in self.graphs or []:
            g.free()
        for p in self.buffers:
            self.ctx.device_free(p)
        self.buffers = []

    # ---- a step
    def _call(self, fn, *args) -> None:
        if fn(self.ctx.handle, *args) != 0:
            raise RuntimeError(si_hip.last_error())

    def _submit(self, which: int) -> None:
        """The device calls of one step on cache `which`."""
        ctx, lib, n, h = self.ctx, self.lib, self.rows, self.hidden
        kv = self.kv_heads * self.head_dim
        cache = self.caches[which]
        norm = lambda x, y: self._call(lib.si_hip_rms_norm_device, 1, x, None, self.norm, n, h, 1e-6, y)  # noqa: E731

        def times(w, rows, x, y):  # (a product takes up to MAX_BATCH rows of x)
            for r in range(0, n, si_hip.MAX_BATCH):
                self._call(lib.si_hip_matmul_many_device, w.handle, rows, h,
                           min(n - r, si_hip.MAX_BATCH), x + 4 * r * h, y + 4 * r * rows)

        self._call(lib.si_hip_embedding_device, self.embed.handle, h, self.vocab, self.d_ids, n, self.d_x)
        norm(self.d_x, self.d_h)
        times(self.w_q, h, self.d_h, self.d_q)
        times(self.w_k, kv, self.d_h, self.d_k)
        times(self.w_v, kv, self.d_h, self.d_v)
        ctx.rope_append_device(cache, self.tokens, self.d_k, self.d_v, rope=self.rope,
                               d_positions=self.d_positions, d_q=self.d_q, heads=self.heads,
                               d_q_out=self.d_q_rot)
        ctx.paged_attention_device(cache, self.heads, self.tokens, self.head_dim ** -0.5,
                                   self.d_q_rot, self.d_attn, self.space, self.space_bytes,
                                   d_weights=self.weights[which], weights_stride=self.capacity)
        times(self.w_o, h, self.d_attn, self.d_o)
        norm(self.d_o, self.d_h)
        times(self.head, self.vocab, self.d_h, self.d_logits)
        ctx.softmax_device(self.d_logits, n, self.vocab, self.temperature, self.d_probs)
        ctx.verify_draft_device(self.d_probs, None, self.d_drafts, self.d_uniform, self.sequences,
                                self.drafts, self.vocab, self.d_accepted, self.d_next)
        # the token that was there and the accepted drafts are part of the sequence now; the
        # others' rows are written over by the next step
        ctx.kv_advance_device(cache, self.d_accepted, 1)

    def _capture(self, which: int):
        self.ctx.capture_begin()
        self._submit(which)
        return self.ctx.capture_end()

    def _evict(self) -> None:
        source, to = self.now, 1 - self.now
        self.ctx.to_device(self.weights[to], np.zeros((self.sequences, self.kv_heads, self.capacity),
                                                      np.float32))
        self.ctx.kv_evict_device(self.caches[source], self.weights[source], self.capacity, self.keep,
                                 self.sinks, self.recent, self.caches[to], self.weights[to],
                                 self.capacity, self.kept)
        self.now = to
        self.lengths = np.minimum(self.lengths, self.keep)
        self.evictions += 1

    def step(self) -> list[list[int]]:
        """One step of every sequence; the tokens that each gained."""
        if self.lengths.max() + self.tokens > self.capacity:
            self._evict()
        proposals = [self.drafter.propose(t, self.drafts) for t in self.text]
        ids = np.array([[t[-1], *p] for t, p in zip(self.text, proposals)], np.uint32)
        # (a cached token keeps the position it was rotated by, whatever is evicted)
        positions = np.array([np.arange(len(t) - 1, len(t) - 1 + self.tokens) for t in self.text],
                             np.uint32)
        self.ctx.to_device(self.d_ids, ids)
        self.ctx.to_device(self.d_positions, positions)
        self.ctx.to_device(self.d_drafts, np.array(proposals, np.uint32))
        self.ctx.to_device(self.d_uniform, self.rng.random((self.sequences, self.drafts + 1),
                                                           dtype=np.float32))
        if self.graphs:
            self.graphs[self.now].launch()
        else:
            self._submit(self.now)
        self.ctx.synchronize()
        accepted = self.ctx.from_device(self.d_accepted, (self.sequences,), np.uint32)
        after = self.ctx.from_device(self.d_next, (self.sequences, self.drafts + 1), np.uint32)
        gained = [[int(x) for x in row[:n + 1]] for row, n in zip(after, accepted)]
        for i, new in enumerate(gained):
            self.text[i].extend(new)
            self.lengths[i] += len(new)
            # the slots of refused drafts are other tokens' next: what they weighed is forgotten
            for h in range(self.kv_heads if len(new) < self.tokens else 0):
                slot = (i * self.kv_heads + h) * self.capacity + int(self.lengths[i])
                self.ctx.to_device(self.weights[self.now] + 4 * slot,
                                   np.zeros(self.tokens - len(new), np.float32))
        return gained


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--sequences", type=int, default=2)
    parser.add_argument("--drafts", type=int, default=3)
    parser.add_argument("--temperature", type=float, default=0.15)
    args = parser.parse_args()
    ctx = si_hip.HipContext(0)
    decoder = SpeculativeDecoder(ctx, sequences=args.sequences, drafts=args.drafts,
                                 temperature=args.temperature)
    made = sum(len(new) for _ in range(args.steps) for new in decoder.step())
    for i, text in enumerate(decoder.text):
        print(f"sequence {i}: {len(text)} tokens, cache {decoder.lengths[i]}: {text[:12]} ...")
    print(f"{made} tokens in {args.steps} steps of {args.sequences} sequences, "
          f"{decoder.evictions} evictions")
    decoder.close()
    ctx.close()


if __name__ == "__main__":
    main()
