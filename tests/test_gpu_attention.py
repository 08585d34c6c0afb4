"""GPU: attention of new tokens over a paged cache against 64-bit arithmetic
(decode_ref.attention derives the tolerance), at the lengths, page sizes, head
layouts and masks where it can go wrong, under both kernel policies."""
import numpy as np
import pytest

import decode_ref as R
import si_hip
from si_hip import HipError

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(hip_ctx):
    d = R.Device(hip_ctx)
    yield d
    hip_ctx.synchronize()
    d.free()


def attend(ctx, dev, c, q, scale, window=0, counts=None, weights=None, gap=0, offset=0):
    b, t, h, d = q.shape
    wide = np.full((b, t, h, d + gap), np.nan, np.float32)
    wide[..., :d] = q
    size = ctx.paged_attention_workspace(c.handle, h, t, weights is not None)
    d_out = dev.put(np.full(q.shape, 9.0, np.float32), offset)
    d_w = None if weights is None else dev.put(weights)
    ctx.paged_attention_device(c.handle, h, t, scale, dev.put(wide, offset), d_out, dev.raw(size),
                               size, window=window,
                               d_counts=None if counts is None else dev.put(counts),
                               q_head_stride=d + gap, d_weights=d_w,
                               weights_stride=0 if weights is None else weights.shape[2])
    ctx.synchronize()
    out = dev.get(d_out, np.empty(q.shape, np.float32))
    return (out, dev.get(d_w, weights)) if weights is not None else out


def check(got, want, tol, what=""):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {np.argwhere(bad)[:3].tolist()} worst {np.nanmax(err / (tol + 1e-30)):.2f}"


def both_policies(ctx):
    yield "tuned"
    ctx.set_kernel_policy(si_hip.KERNEL_GENERIC)
    try:
        yield "generic"
    finally:
        ctx.set_kernel_policy(si_hip.KERNEL_AUTO)


def run(ctx, dev, c, q, window=0, counts=None, weights=False, gap=0, offset=0, scale=None, what=""):
    scale = scale or q.shape[3] ** -0.5
    scale = float(np.float32(scale))
    want, tol, w, wtol = R.attention(c, q, scale, window, counts)
    if weights:
        old = np.random.default_rng(5).random((q.shape[0], c.kv_heads, c.capacity + 3)).astype(np.float32)
    for policy in both_policies(ctx):
        if not weights:
            check(attend(ctx, dev, c, q, scale, window, counts, None, gap, offset), want, tol,
                  f"{policy} {what}")
            continue
        out, got = attend(ctx, dev, c, q, scale, window, counts, old, gap, offset)
        check(out, want, tol, f"{policy} {what}")
        n = c.capacity
        # the sum and the addition to what was there round once more each
        check(got[..., :n], old[..., :n] + w, wtol + 2.0 ** -23 * (old[..., :n] + w),
              f"{policy} weights {what}")
        untouched = w == 0
        assert np.array_equal(got[..., :n][untouched], old[..., :n][untouched])
        assert np.array_equal(got[..., n:], old[..., n:])


LENGTHS = [0, 1, 2, 15, 16, 17, 30, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300, 511, 700]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (6, 1, 256), (4, 4, 64), (5, 1, 96), (14, 2, 80),
                                          (2, 2, 192), (40, 2, 32), (3, 3, 8), (2, 1, 40)])
def test_lengths_and_heads(hip_ctx, dev, kind, heads, kv, dim):
    rng = np.random.default_rng(heads * 1000 + dim)
    c = R.Cache(dev, rng, kind, len(LENGTHS), kv, dim, 16, 45, LENGTHS)
    q = (rng.standard_normal((len(LENGTHS), 1, heads, dim)) * 2).astype(np.float32)
    run(hip_ctx, dev, c, q)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [1, 7, 33, 50, 100, 250])
def test_odd_head_sizes(hip_ctx, dev, kind, dim):
    rng = np.random.default_rng(dim)
    c = R.Cache(dev, rng, kind, 3, 2, dim, 16, 8, [0, 40, 126])
    run(hip_ctx, dev, c, rng.standard_normal((3, 2, 6, dim)).astype(np.float32))


@pytest.mark.parametrize("page", [1, 2, 3, 4, 5, 8, 24, 32, 33, 64, 100, 128])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_page_sizes(hip_ctx, dev, page, kind):
    rng = np.random.default_rng(page)
    lengths = [0, 3, 29, 150, 333]
    c = R.Cache(dev, rng, kind, 5, 2, 64, page, -(-340 // page), lengths)
    run(hip_ctx, dev, c, rng.standard_normal((5, 3, 4, 64)).astype(np.float32))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 8, 13, 16])
@pytest.mark.parametrize("heads,kv,dim", [(6, 1, 256), (8, 2, 128), (1, 1, 64), (32, 1, 64)])
def test_several_tokens(hip_ctx, dev, kind, tokens, heads, kv, dim):
    rng = np.random.default_rng(tokens * 10 + dim)
    lengths = [0, 1, 31, 64, 201]
    c = R.Cache(dev, rng, kind, 5, kv, dim, 16, 14, lengths)
    q = rng.standard_normal((5, tokens, heads, dim)).astype(np.float32)
    run(hip_ctx, dev, c, q, weights=True)
    counts = np.array([tokens, 0, 1, tokens // 2, 0xFFFFFFFF], np.uint32)
    run(hip_ctx, dev, c, q, counts=counts, weights=True, what="counts")


@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 100, 1000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_windows(hip_ctx, dev, window, kind):
    rng = np.random.default_rng(window)
    lengths = [0, 5, 32, 99, 400, 517]
    c = R.Cache(dev, rng, kind, 6, 2, 128, 16, 34, lengths)
    q = rng.standard_normal((6, 5, 4, 128)).astype(np.float32)
    run(hip_ctx, dev, c, q, window=window, weights=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,offset", [(64, 4), (128, 8), (256, 2), (128, 16)])
def test_alignments_and_strides(hip_ctx, dev, kind, dim, offset):
    if offset % (4 if kind == "f32" else 2):
        pytest.skip("not an address of this type")
    rng = np.random.default_rng(offset)
    c = R.Cache(dev, rng, kind, 3, 2, dim, 16, 10, [7, 64, 150], offset=offset)
    q = rng.standard_normal((3, 2, 6, dim)).astype(np.float32)
    run(hip_ctx, dev, c, q, gap=5, offset=4)
    run(hip_ctx, dev, c, q, gap=dim, weights=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads", [4, 10, 16])  # one, two and three row tiles
def test_numbers_in_unseen_slots_do_not_matter(hip_ctx, dev, kind, dim, heads):
    """NaN and infinities behind the sequence, before the window, in later new
    tokens' rows for the earlier ones, and on pages of nobody."""
    rng = np.random.default_rng(dim)
    lengths, tokens, window = [0, 21, 90, 150], 6, 40
    c = R.Cache(dev, rng, kind, 4, 2, dim, 16, 11, lengths)
    clean = R.attention(c, q := rng.standard_normal((4, tokens, heads, dim)).astype(np.float32),
                        float(np.float32(dim ** -0.5)), window, None)
    seen = np.zeros(c.keys.shape[:3:2], bool)  # [page][place]
    for s, n in enumerate(lengths):
        for slot in range(max(0, n + 1 - window), n + tokens):
            seen[c.at(s, slot)] = True
    for bad in (np.nan, np.inf, -np.inf):
        k, v = R.decode(c.keys, kind).copy(), R.decode(c.values, kind).copy()
        for a in (k, v):
            a.transpose(0, 2, 1, 3)[~seen] = bad
        old = c.keys, c.values
        c.keys, c.values = R.encode(k, kind), R.encode(v, kind)
        c.upload()
        for policy in both_policies(hip_ctx):
            check(attend(hip_ctx, dev, c, q, dim ** -0.5, window), clean[0], clean[1], f"{policy} {bad}")
        c.keys, c.values = old
    # the last new token's own row: only its own output may see it
    v = R.decode(c.values, kind).copy()
    k = R.decode(c.keys, kind).copy()
    for s, n in enumerate(lengths):
        p, o = c.at(s, n + tokens - 1)
        v[p, :, o] = np.nan
        k[p, :, o, 0] = np.inf
    c.keys, c.values = R.encode(k, kind), R.encode(v, kind)
    c.upload()
    for policy in both_policies(hip_ctx):
        out = attend(hip_ctx, dev, c, q, dim ** -0.5, window)
        check(out[:, :-1], clean[0][:, :-1], clean[1][:, :-1], f"{policy} later token")
        assert np.isnan(out[:, -1]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_large_and_small_scores(hip_ctx, dev, kind):
    """Scores far apart, a first slot that outweighs all others, rows of zeros, and query
    values from the smallest to the largest that the products can hold."""
    rng = np.random.default_rng(11)
    c = R.Cache(dev, rng, kind, 4, 2, 128, 16, 20, [40, 130, 300, 310])
    q = rng.standard_normal((4, 1, 4, 128)).astype(np.float32)
    q[0] *= 100.0
    q[1] = 0.0
    q[2] *= 1e-30
    q[3, 0, 0] *= 1e4
    q[3, 0, 1, 5] = 3e5
    run(hip_ctx, dev, c, q, weights=True)
    run(hip_ctx, dev, c, q, scale=-0.1)
    run(hip_ctx, dev, c, np.abs(q).clip(max=1e3) * 1e30, scale=1e-31)


def test_idle_and_invalid_sequences(hip_ctx, dev):
    rng = np.random.default_rng(12)
    q = rng.standard_normal((3, 2, 4, 64)).astype(np.float32)
    for kind in ("f32", "f16", "bf16"):
        c = R.Cache(dev, rng, kind, 3, 2, 64, 16, 4, [20, 60, 33])
        c.table[0, 0] = 0xFFFFFFFF  # the first sixteen slots lie nowhere
        c.table[2] = c.keys.shape[0]  # nothing of this one does
        c.upload()
        want, tol, _, _ = R.attention(c, q, 0.125, 0, None)
        assert not want[2].any()
        for policy in both_policies(hip_ctx):
            size = hip_ctx.paged_attention_workspace(c.handle, 4, 2)
            d_out = dev.put(np.full(q.shape, 9.0, np.float32))
            hip_ctx.paged_attention_device(c.handle, 4, 2, 0.125, dev.put(q), d_out, dev.raw(size), size)
            with pytest.raises(HipError) as e:
                hip_ctx.synchronize()
            assert "pool" in e.value.message
            check(dev.get(d_out, q), want, tol, f"{kind} {policy}")
        # more tokens than the pages hold
        c = R.Cache(dev, rng, kind, 3, 2, 64, 16, 4, [20, 63, 0xFFFFFFFF])
        want, tol, _, _ = R.attention(c, q, 0.125, 0, None)
        for policy in both_policies(hip_ctx):
            size = hip_ctx.paged_attention_workspace(c.handle, 4, 2)
            d_out = dev.put(np.full(q.shape, 9.0, np.float32))
            hip_ctx.paged_attention_device(c.handle, 4, 2, 0.125, dev.put(q), d_out, dev.raw(size), size)
            with pytest.raises(HipError) as e:
                hip_ctx.synchronize()
            assert "do not fit" in e.value.message
            check(dev.get(d_out, q), want, tol, f"{kind} {policy}")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_long_sequences_split_and_join(hip_ctx, dev, kind):
    """Few rows over many slots, several sequences of very different lengths,
    and the same call again: its result does not depend on timing."""
    rng = np.random.default_rng(13)
    lengths = [40000, 3, 9001, 0]
    c = R.Cache(dev, rng, kind, 4, 1, 64, 64, 626, lengths)
    q = (rng.standard_normal((4, 2, 2, 64)) * 2).astype(np.float32)
    want, tol, _, _ = R.attention(c, q, 0.125, 0, None)
    # the sums' walk over 40000 slots instead of 4096
    tol = tol + 200 * 2.0 ** -24 * np.abs(tol) / 2.0 ** -20
    first = attend(hip_ctx, dev, c, q, 0.125)
    check(first, want, tol)
    for _ in range(4):
        assert np.array_equal(attend(hip_ctx, dev, c, q, 0.125), first)


def test_many_sequences(hip_ctx, dev):
    rng = np.random.default_rng(14)
    lengths = rng.integers(0, 120, 333)
    c = R.Cache(dev, rng, "f16", 333, 2, 64, 8, 16, lengths)
    run(hip_ctx, dev, c, rng.standard_normal((333, 1, 4, 64)).astype(np.float32), weights=True)


@pytest.mark.parametrize("sequences", [2, 3, 17, 63, 64, 65, 130])
@pytest.mark.parametrize("kind,heads,dim,tokens", [("f16", 2, 64, 1), ("bf16", 3, 256, 7), ("f32", 2, 128, 9)])
def test_shares_end_anywhere(hip_ctx, dev, kind, heads, dim, tokens, sequences):
    """Batches of lengths from none to many rounds: shares that begin and end
    inside sequences, between them, and over several of them."""
    rng = np.random.default_rng(sequences)
    lengths = np.where(rng.random(sequences) < 0.3, rng.integers(800, 3500, sequences),
                       rng.integers(0, 300, sequences))
    c = R.Cache(dev, rng, kind, sequences, 1, dim, 16, 3520 // 16, lengths)
    counts = rng.integers(0, tokens + 1, sequences).astype(np.uint32)
    q = rng.standard_normal((sequences, tokens, heads, dim)).astype(np.float32)
    run(hip_ctx, dev, c, q, weights=sequences in (3, 65), counts=counts)


def test_cache_beyond_four_gigabytes(hip_ctx, dev):
    """Pages at both ends of a pool of more than 2^32 values."""
    kv, dim, page = 1, 128, 64
    pages = (1 << 32) // (kv * dim * page) + 70
    nbytes = pages * kv * dim * page * 2
    keys, values = dev.raw(nbytes), dev.raw(nbytes)
    rng = np.random.default_rng(15)
    c = R.Cache(dev, rng, "f16", 1, kv, dim, page, 6, [333])
    table = np.array([[pages - 1, 0, pages - 40, 1, pages - 69, pages - 2]], np.uint32)
    for i, p in enumerate(table[0]):
        n = kv * page * dim * 2
        dev.ctx.to_device(keys + int(p) * n, c.keys[c.table[0, i]])
        dev.ctx.to_device(values + int(p) * n, c.values[c.table[0, i]])
    q = rng.standard_normal((1, 2, 4, dim)).astype(np.float32)
    want, tol, _, _ = R.attention(c, q, 0.1, 0, None)
    c.handle.d_keys, c.handle.d_values, c.handle.pages = keys, values, pages
    c.handle.d_page_table = dev.put(table)
    for policy in both_policies(hip_ctx):
        check(attend(hip_ctx, dev, c, q, 0.1), want, tol, policy)


def test_captured_steps(hip_ctx, dev):
    """Append, attention with weights and advance in one graph: each replay is
    the next decode step."""
    rng = np.random.default_rng(16)
    c = R.Cache(dev, rng, "bf16", 2, 2, 128, 16, 6, [30, 61])
    table, magnitude = si_hip.rope_frequencies(64, 1e6)
    inv, _ = R.inverse_frequencies(64, 1e6)
    rope = si_hip.Rope(layout=1, rotary_dim=64, magnitude=magnitude, d_frequencies=dev.put(table))
    q, k, v = (rng.standard_normal((2, 1, n, 128)).astype(np.float32) for n in (8, 2, 2))
    d = {n: dev.put(x) for n, x in (("q", q), ("k", k), ("v", v))}
    d_q, d_out = dev.put(np.zeros_like(q)), dev.put(np.zeros_like(q))
    weights = np.zeros((2, 2, c.capacity), np.float32)
    d_w = dev.put(weights)
    size = hip_ctx.paged_attention_workspace(c.handle, 8, 1, True)
    space = dev.raw(size)
    hip_ctx.capture_begin()
    hip_ctx.rope_append_device(c.handle, 1, d["k"], d["v"], rope=rope, d_q=d["q"], heads=8, d_q_out=d_q)
    hip_ctx.paged_attention_device(c.handle, 8, 1, 0.1, d_q, d_out, space, size, d_weights=d_w,
                                   weights_stride=c.capacity)
    hip_ctx.kv_advance_device(c.handle, None, 1)
    graph = hip_ctx.capture_end()
    assert graph.calls == 3
    total, total_tol = np.zeros((2, 2, c.capacity)), np.zeros((2, 2, c.capacity))
    for step in range(5):
        graph.launch()
        hip_ctx.synchronize()
        c.keys, c.values = c.device("keys"), c.device("values")
        qr, _ = R.rotate(q[:, 0], c.lengths, inv, 1.0, 1)
        got_q = dev.get(d_q, q)
        assert np.abs(got_q[:, 0] - qr).max() < 1e-5
        want, tol, w, wtol = R.attention(c, got_q, float(np.float32(0.1)), 0, None)
        check(dev.get(d_out, q), want, tol, f"step {step}")
        total, total_tol = total + w, total_tol + wtol + 2.0 ** -23 * (total + w)
        check(dev.get(d_w, weights), total, total_tol, f"weights {step}")
        c.lengths = c.lengths + 1
        assert np.array_equal(dev.get(c.d_lengths, c.lengths), c.lengths)


def test_weights_of_a_capacity_beyond_one_launch(hip_ctx, dev):
    """Weights of a table of 2^30 slots, few of them in use: four workgroups of 64 threads each
    for 64 slots are more threads than a launch takes."""
    rng = np.random.default_rng(17)
    c = R.Cache(dev, rng, "f16", 1, 1, 64, 16, 20, [300])
    tokens, heads = 5, 2
    q = rng.standard_normal((1, tokens, heads, 64)).astype(np.float32)
    want, tol, w, wtol = R.attention(c, q, 0.125, 0, None)
    c.handle.max_pages = (1 << 26) + 1
    table = dev.raw(4 * c.handle.max_pages)
    dev.ctx.to_device(table, c.table)
    c.handle.d_page_table = table
    capacity = c.handle.capacity
    d_w = dev.raw(4 * capacity)
    old = rng.random((1, 1, c.capacity)).astype(np.float32)
    dev.ctx.to_device(d_w, old)
    size = hip_ctx.paged_attention_workspace(c.handle, heads, tokens, True)
    d_out = dev.put(np.full(q.shape, 9.0, np.float32))
    hip_ctx.paged_attention_device(c.handle, heads, tokens, 0.125, dev.put(q), d_out, dev.raw(size),
                                   size, d_weights=d_w, weights_stride=capacity)
    hip_ctx.synchronize()
    check(dev.get(d_out, q), want, tol)
    check(dev.get(d_w, old), old + w, wtol + 2.0 ** -23 * (old + w))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim", [(4, 128), (20, 128), (4, 256), (20, 256), (4, 80)])
def test_one_query_value_far_above_the_others(hip_ctx, dev, kind, heads, dim):
    """Where the keys are zero beside it, the others alone make the scores.  They lie down to
    2^-28 of it, where an F16 cache's calls hold 22 bits of them: 2 units in the last place
    of sum |q k| at most, within the 16 of the tolerance."""
    rng = np.random.default_rng(heads + dim)
    c = R.Cache(dev, rng, kind, 3, 2, dim, 16, 14, [200, 33, 7])
    c.keys[..., 0] = 0
    c.keys[..., dim - 1] = 0
    c.upload()
    q = rng.uniform(1.0, 2.0, (3, 2, heads, dim)) * rng.choice([-1.0, 1.0], (3, 2, heads, dim))
    q[:, 0, :, 0] = 2.0 ** 28
    q[:, 1, :, dim - 1] = -2.0 ** 20
    run(hip_ctx, dev, c, q.astype(np.float32), weights=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim", [(4, 128), (20, 128), (20, 256), (4, 80)])
@pytest.mark.parametrize("bits", [12, 24, 34])
def test_weights_far_below_the_largest(hip_ctx, dev, kind, heads, dim, bits):
    """A first slot that outweighs each other one 2^bits times, with values of 0: the others
    alone make the output.  An F16 cache's calls hold their p to 2^-39 of the largest."""
    rng = np.random.default_rng(heads + dim + bits)
    c = R.Cache(dev, rng, kind, 3, 2, dim, 16, 14, [200, 33, 7])
    scale = float(np.float32(dim ** -0.5))
    c.keys = R.encode(R.decode(c.keys, kind) * 0.1, kind)
    for s in range(3):
        p, o = c.at(s, 0)
        c.keys[p, :, o] = R.encode(np.full(dim, bits * np.log(2.0) / (scale * dim)), kind)
        c.values[p, :, o] = 0
    c.upload()
    q = rng.uniform(0.98, 1.02, (3, 2, heads, dim)).astype(np.float32)
    want, tol, _, _ = R.attention(c, q, scale, 0, None)
    assert np.all(np.abs(want) < 200 * 8 * 2.0 ** -(0.9 * bits))
    if kind == "f16":
        for s, n in enumerate(c.lengths):
            for kv in range(2):
                v = np.abs(c.rows("values", s, kv, np.arange(int(n) + 2))).sum(0)
                tol[s, :, kv * heads // 2:(kv + 1) * heads // 2] += 2.0 ** -39 * v
    for policy in both_policies(hip_ctx):
        check(attend(hip_ctx, dev, c, q, scale), want, tol, policy)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 32])
@pytest.mark.parametrize("heads,dim,tokens", [(4, 64, 1), (20, 128, 3), (12, 256, 5), (6, 80, 3)])
def test_pages_behind_the_window(hip_ctx, dev, kind, page, heads, dim, tokens):
    """A page that no row sees any more may lie anywhere; one with a seen slot is reported."""
    window = 40
    rng = np.random.default_rng(page * 1000 + dim)
    c = R.Cache(dev, rng, kind, 4, 2, dim, page, -(-320 // page), [100, 61, 300, 12])
    for s, n in enumerate(c.lengths):
        c.table[s, :max(0, int(n) + 1 - window) // page] = 0xFFFFFFFF
    assert (c.table[0, 0] == 0xFFFFFFFF) and c.table[3, 0] != 0xFFFFFFFF
    c.upload()
    q = rng.standard_normal((4, tokens, heads, dim)).astype(np.float32)
    run(hip_ctx, dev, c, q, window=window, weights=True)
    c.table[2, (301 - window) // page] = 0xFFFFFFFF  # the one with the first slot that is seen
    c.upload()
    scale = float(np.float32(dim ** -0.5))
    want, tol, _, _ = R.attention(c, q, scale, window, None)
    for policy in both_policies(hip_ctx):
        size = hip_ctx.paged_attention_workspace(c.handle, heads, tokens)
        d_out = dev.put(np.full(q.shape, 9.0, np.float32))
        hip_ctx.paged_attention_device(c.handle, heads, tokens, scale, dev.put(q), d_out,
                                       dev.raw(size), size, window=window)
        with pytest.raises(HipError) as e:
            hip_ctx.synchronize()
        assert "pool" in e.value.message
        check(dev.get(d_out, q), want, tol, policy)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_long_sequences_within_their_sums_walk(hip_ctx, dev, kind):
    rng = np.random.default_rng(13)
    c = R.Cache(dev, rng, kind, 4, 1, 64, 64, 626, [40000, 3, 9001, 0])
    q = (rng.standard_normal((4, 2, 2, 64)) * 2).astype(np.float32)
    want, tol, _, _ = R.attention(c, q, 0.125, 0, None, walk=40002)
    for policy in both_policies(hip_ctx):
        check(attend(hip_ctx, dev, c, q, 0.125), want, tol, policy)


@pytest.mark.parametrize("kind,dim,heads,tokens,slots", [
    ("bf16", 256, 2, 1, 20000), ("f16", 256, 6, 7, 20000), ("f32", 256, 3, 4, 12000),
    ("f32", 128, 2, 2, 20000), ("bf16", 128, 4, 1, 40000), ("f16", 128, 8, 4, 40000)])
def test_a_sequence_in_more_shares_than_the_join_loads_at_once(hip_ctx, dev, kind, dim, heads, tokens,
                                                               slots):
    """One kv head of one sequence is dealt to some hundred workgroups; a thread of the join holds
    eight shares of a head of 256 in each of eight groups, or of 128 in sixteen, and takes the
    others one by one.  Its result, weights too, does not depend on timing."""
    rng = np.random.default_rng(slots + dim)
    c = R.Cache(dev, rng, kind, 1, 1, dim, 16, (slots + tokens + 15) // 16, [slots])
    q = (rng.standard_normal((1, tokens, heads, dim)) * 2).astype(np.float32)
    scale = float(np.float32(dim ** -0.5))
    want, tol, w, wtol = R.attention(c, q, scale, 0, None, walk=slots)
    zero = np.zeros((1, 1, c.capacity), np.float32)
    first, weights = attend(hip_ctx, dev, c, q, scale, weights=zero)
    check(first, want, tol)
    check(weights, w, wtol)
    for _ in range(3):
        again, once_more = attend(hip_ctx, dev, c, q, scale, weights=zero)
        assert np.array_equal(again, first) and np.array_equal(once_more, weights)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,group,dim,tokens,lengths", [
    (32, 1, 64, 1, [2047]),             # eight shares of one sequence
    (32, 2, 128, 2, [1500, 40, 700]),   # shares that end in sequences and between them
    (40, 1, 256, 1, [600, 0, 333]),
    (100, 1, 128, 1, [900, 500]),       # two shares
    (32, 3, 64, 9, [1100, 200]),        # two row tiles at once
    (32, 3, 256, 15, [700, 90]),        # three
    (16, 5, 128, 16, [800, 100]),       # several groups of them
    (33, 2, 80, 1, [1000, 513]), (12, 6, 80, 7, [900])])
def test_shares_joined_by_the_last_of_them(hip_ctx, dev, kind, kv, group, dim, tokens, lengths):
    """Many kv heads leave few shares a sequence; the last one that is done joins them.  Call after
    call, with and without weights, the counters are back where they were."""
    rng = np.random.default_rng(kv + dim)
    heads = kv * group
    c = R.Cache(dev, rng, kind, len(lengths), kv, dim, 16, (max(lengths) + tokens + 15) // 16, lengths)
    q = rng.standard_normal((len(lengths), tokens, heads, dim)).astype(np.float32)
    scale = float(np.float32(dim ** -0.5))
    want, tol, w, wtol = R.attention(c, q, scale, 0, None)
    zero = np.zeros((len(lengths), kv, c.capacity), np.float32)
    first, weights = attend(hip_ctx, dev, c, q, scale, weights=zero)
    check(first, want, tol)
    check(weights, w, wtol)
    assert np.array_equal(attend(hip_ctx, dev, c, q, scale), first)
    # fewer tokens and a window: other sequences are split, or none
    counts = np.arange(len(lengths), dtype=np.uint32) % (tokens + 1)
    want, tol, _, _ = R.attention(c, q, scale, 300, counts)
    check(attend(hip_ctx, dev, c, q, scale, window=300, counts=counts), want, tol)
    for _ in range(3):
        again, once_more = attend(hip_ctx, dev, c, q, scale, weights=zero)
        assert np.array_equal(again, first) and np.array_equal(once_more, weights)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(10, 2, 80, 16), (6, 1, 96, 32), (8, 2, 192, 16),
                                               (10, 2, 64, 24), (5, 1, 128, 7), (6, 2, 256, 40)])
def test_several_row_tiles_at_any_address(hip_ctx, dev, kind, heads, kv, dim, page):
    rng = np.random.default_rng(heads + dim + page)
    lengths = [0, 17, 130, 401, 64]
    c = R.Cache(dev, rng, kind, 5, kv, dim, page, -(-420 // page), lengths)
    q = rng.standard_normal((5, 11, heads, dim)).astype(np.float32)
    run(hip_ctx, dev, c, q, weights=True)
    counts = np.array([11, 4, 0, 9, 1], np.uint32)
    run(hip_ctx, dev, c, q, window=100, counts=counts, weights=True, what="counts")
