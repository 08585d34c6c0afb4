"""GPU: the speculative decoding example: each step's attention, probabilities
and tokens against the CPU references on the step's own inputs, replayed from
graphs and submitted call by call, through evictions."""
import sys
from pathlib import Path

import numpy as np
import pytest

import decode_ref as R

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


class HostCache:
    """The decoder's present cache as decode_ref sees one."""

    def __init__(self, d, which, kind):
        c = d.caches[which]
        shape = (c.pages, c.kv_heads, c.page_tokens, c.head_dim)
        dtype = R.TYPES[kind][1]
        self.kind, self.page, self.max_pages = kind, c.page_tokens, c.max_pages
        self.kv_heads, self.head_dim = c.kv_heads, c.head_dim
        self.keys = d.ctx.from_device(c.d_keys, shape, dtype)
        self.values = d.ctx.from_device(c.d_values, shape, dtype)
        self.table = d.page_tables[which]
        self.lengths = np.zeros(c.sequences, np.uint32)

    capacity = R.Cache.capacity
    rows = R.Cache.rows
    at = R.Cache.at


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_every_step(hip_ctx, kind):
    from speculative_decode import SpeculativeDecoder
    decoders = [SpeculativeDecoder(hip_ctx, cache_type=R.TYPES[kind][0], use_graph=g)
                for g in (True, False)]
    d = decoders[0]
    total = np.zeros((2, d.sequences, d.kv_heads, d.capacity))
    total_tol = np.zeros_like(total)
    for step in range(80):
        before, was = d.lengths.copy(), d.now
        texts = [list(t) for t in d.text]
        gained = d.step()
        assert gained == decoders[1].step()  # the same numbers, call by call
        if d.now != was:  # evicted: each head's weights went with its slots
            kept = d.ctx.from_device(d.kept, (d.sequences, d.kv_heads, d.keep), np.uint32)
            moved, moved_tol = np.zeros_like(total[0]), np.zeros_like(total[0])
            for s in range(d.sequences):
                n = min(before[s], d.keep)
                assert np.all(kept[s, :, n:] == R.NONE)
                for h in range(d.kv_heads):
                    slots = kept[s, h, :n].astype(int)
                    assert np.all(np.diff(slots) > 0) and slots[-1] < before[s]
                    if before[s] > d.keep:
                        assert np.array_equal(slots[:d.sinks], np.arange(d.sinks))
                        assert np.array_equal(slots[-d.recent:],
                                              np.arange(before[s] - d.recent, before[s]))
                    moved[s, h, :n], moved_tol[s, h, :n] = total[was, s, h, slots], total_tol[was, s, h, slots]
            total[d.now], total_tol[d.now] = moved, moved_tol
            before = np.minimum(before, d.keep)
        c = HostCache(d, d.now, kind)
        c.lengths = before.astype(np.uint32)
        q = d.ctx.from_device(d.d_q_rot, (d.sequences, d.tokens, d.heads, d.head_dim))
        out = d.ctx.from_device(d.d_attn, q.shape)
        want, tol, w, wtol = R.attention(c, q, float(np.float32(d.head_dim ** -0.5)), 0, None)
        assert np.all(np.abs(out - want) <= tol), f"step {step}"
        total[d.now] += w
        total_tol[d.now] += wtol + 2.0 ** -23 * total[d.now]
        for s in range(d.sequences):  # refused drafts leave nothing in their slots
            total[d.now, s, :, before[s] + len(gained[s]):] = 0.0
        got = d.ctx.from_device(d.weights[d.now], w.shape)
        assert np.all(np.abs(got - total[d.now]) <= total_tol[d.now] + 1e-30), f"step {step}"
        # the tokens from the step's probabilities
        p = d.ctx.from_device(d.d_probs, (d.sequences, d.tokens, d.vocab))
        assert np.allclose(p.sum(2, dtype=np.float64), 1.0, atol=1e-5)
        u = d.ctx.from_device(d.d_uniform, (d.sequences, d.drafts + 1))
        drafts = d.ctx.from_device(d.d_drafts, (d.sequences, d.drafts), np.uint32)
        accepted, tokens = R.verify(p, None, drafts, None, u, d.vocab)
        for s in range(d.sequences):
            assert gained[s] == [int(x) for x in tokens[s, :accepted[s] + 1]]
            assert d.text[s] == texts[s] + gained[s]
        held = d.ctx.from_device(d.caches[d.now].d_lengths, (d.sequences,), np.uint32)
        assert np.array_equal(held, before + accepted + 1) and np.array_equal(held, d.lengths)
    assert d.evictions >= 1
    for x in decoders:
        x.close()


def test_more_rows_than_one_product_takes(hip_ctx):
    """Five sequences of four rows: products of sixteen rows and of four.  A row's logits are its
    own: both are far closer than 2^-15 of |w| |h| to the product, another row's lie about |w| |h|
    / 20 away."""
    from speculative_decode import SpeculativeDecoder
    decoders = [SpeculativeDecoder(hip_ctx, sequences=5, use_graph=g) for g in (True, False)]
    d = decoders[0]
    for _ in range(30):
        gained = d.step()
        assert gained == decoders[1].step()
        h = d.ctx.from_device(d.d_h, (d.rows, d.hidden))
        logits = d.ctx.from_device(d.d_logits, (d.rows, d.vocab))
        for r in (0, 15, 16, 19):
            alone = hip_ctx.gguf_quant_matvec_weight(d.head, d.vocab, d.hidden, h[r])
            assert np.abs(logits[r] - alone).max() <= 2.0 ** -15 * 1.1 * np.linalg.norm(h[r])
        p = d.ctx.from_device(d.d_probs, (d.sequences, d.tokens, d.vocab))
        u = d.ctx.from_device(d.d_uniform, (d.sequences, d.drafts + 1))
        drafts = d.ctx.from_device(d.d_drafts, (d.sequences, d.drafts), np.uint32)
        accepted, tokens = R.verify(p, None, drafts, None, u, d.vocab)
        assert gained == [[int(x) for x in t[:a + 1]] for t, a in zip(tokens, accepted)]
    for x in decoders:
        x.close()
