"""GPU: rotary positions and the cache append against 64-bit arithmetic.

Tolerance of a rotated value: its pair's |a| + |b|, times the magnitude, times
5e-7.  The phase, at most half a turn, is rounded to 32 bits (2^-26 of a turn,
9.4e-8 radians), sine and cosine are good to two units in the last place
(1.2e-7), and the magnitude, the product and the sum round once each (6e-8).
"""
import numpy as np
import pytest

import decode_ref as R
import si_hip
from si_hip import HipError

pytestmark = pytest.mark.gpu
REL = 5e-7


@pytest.fixture
def dev(hip_ctx):
    d = R.Device(hip_ctx)
    yield d
    hip_ctx.synchronize()
    d.free()


def make_rope(dev, n, theta=1e6, scaling="none", layout=0):
    code = ("none", "linear", "yarn").index(scaling)
    table, magnitude = si_hip.rope_frequencies(n, theta, code, 4.0, 32768.0)
    inv, m64 = R.inverse_frequencies(n, theta, scaling)
    return si_hip.Rope(layout=layout, rotary_dim=n, magnitude=magnitude,
                       d_frequencies=dev.put(table)), inv, np.float64(np.float32(m64))


def check(got, want, size, what=""):
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= REL * size + 1e-30), f"{what}: {np.max(err / (REL * size + 1e-30)):.3f}"


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dim,n,scaling", [(128, 128, "none"), (256, 64, "linear"), (64, 64, "yarn"),
                                           (80, 40, "none"), (96, 2, "none"), (33, 10, "yarn"),
                                           (2, 2, "none"), (128, 12, "linear")])
def test_rope(hip_ctx, dev, layout, dim, n, scaling):
    rng = np.random.default_rng(dim * 7 + n + layout)
    for tokens, heads, pad, offset in [(1, 1, 0, 0), (5, 3, 0, 0), (37, 7, 4, 0), (3, 5, 1, 4)]:
        rope, inv, mag = make_rope(dev, n, 1e6, scaling, layout)
        x = rng.standard_normal((tokens, heads, dim + pad)).astype(np.float32)
        pos = rng.integers(0, 1 << 20, tokens).astype(np.uint32)
        pos[0] = 0
        if tokens > 2:
            pos[1:3] = [(1 << 32) - 1, 1 << 31]
        want, size = R.rotate(x[..., :dim], pos, inv, mag, layout)
        d_x, d_p = dev.put(x, offset), dev.put(pos)
        d_y = dev.put(np.full((tokens, heads, dim), 7.0, np.float32), offset)
        hip_ctx.rope_device(rope, d_x, tokens, heads, dim, d_p, d_y, head_stride=dim + pad)
        hip_ctx.synchronize()
        # beyond 2^20 positions the f64 reference's angle is itself off by pos * 2^-53 radians
        check(dev.get(d_y, want.astype(np.float32)), want, size + 1e-8, f"{tokens}x{heads}")
        hip_ctx.rope_device(rope, d_x, tokens, heads, dim, d_p, d_x, head_stride=dim + pad,
                            y_head_stride=dim + pad)
        hip_ctx.synchronize()
        got = dev.get(d_x, x)
        check(got[..., :dim], want, size + 1e-8, "in place")
        assert np.array_equal(got[..., dim:], x[..., dim:])  # what lies between rows


def ulp(kind):
    return {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,dim,kv,offset", [(16, 128, 4, 0), (7, 64, 2, 0), (1, 80, 3, 0),
                                                (24, 33, 2, 0), (16, 256, 1, 8), (5, 10, 2, 0)])
def test_append(hip_ctx, dev, kind, page, dim, kv, offset):
    rng = np.random.default_rng(page * 131 + dim)
    for tokens, positions, counts in [(1, True, False), (5, False, True), (3 * page + 2, True, True)]:
        max_pages = -(-(tokens + 40) // page)
        lengths = [0, 17, max_pages * page - tokens]
        c = R.Cache(dev, rng, kind, 3, kv, dim, page, max_pages, lengths, offset)
        rope, inv, mag = make_rope(dev, dim // 2 * 2, 1e4)
        heads, gap = 2 * kv, 3
        k = rng.standard_normal((3 * tokens, kv * dim + gap)).astype(np.float32)
        v = rng.standard_normal((3 * tokens, kv * dim + gap)).astype(np.float32)
        q = rng.standard_normal((3 * tokens, heads, 2 * dim)).astype(np.float32)
        pos = rng.integers(0, 200000, 3 * tokens).astype(np.uint32) if positions else None
        num = np.array([tokens, 0, tokens - 1], np.uint32) if counts else None
        slots = (np.asarray(lengths)[:, None] + np.arange(tokens)).reshape(-1)
        at = pos if positions else slots
        qw, qs = R.rotate(q[..., :dim], at, inv, mag, 0)
        kw, ks = R.rotate(k[:, :kv * dim].reshape(-1, kv, dim), at, inv, mag, 0)
        d_qo = dev.put(np.full((3 * tokens, heads, dim), 5.0, np.float32))
        hip_ctx.rope_append_device(
            c.handle, tokens, dev.put(k), dev.put(v), rope=rope,
            d_counts=None if num is None else dev.put(num),
            d_positions=None if pos is None else dev.put(pos), k_token_stride=kv * dim + gap,
            v_token_stride=kv * dim + gap, d_q=dev.put(q), heads=heads, q_head_stride=2 * dim,
            d_q_out=d_qo)
        hip_ctx.synchronize()
        keys, values = c.device("keys"), c.device("values")
        q_out = dev.get(d_qo, np.empty((3 * tokens, heads, dim), np.float32))
        wk, wv = c.keys.copy(), c.values.copy()
        for s in range(3):
            for t in range(tokens):
                row = s * tokens + t
                if num is not None and t >= num[s]:
                    assert np.all(q_out[row] == 5.0)
                    continue
                p, o = c.at(s, lengths[s] + t)
                got = R.decode(keys[p, :, o], kind)
                err = np.abs(got - kw[row])
                assert np.all(err <= REL * ks[row] + ulp(kind) * np.abs(kw[row]) + 2.0 ** -24)
                assert np.array_equal(values[p, :, o],
                                      R.encode(v[row, :kv * dim].reshape(kv, dim), kind))
                check(q_out[row], qw[row], qs[row], "query")
                wk[p, :, o], wv[p, :, o] = keys[p, :, o], values[p, :, o]
        # every other row of the pool is as it was
        assert np.array_equal(keys, wk) and np.array_equal(values, wv)
        assert np.array_equal(dev.get(c.d_lengths, c.lengths), c.lengths)


def test_append_without_rotation(hip_ctx, dev):
    rng = np.random.default_rng(1)
    c = R.Cache(dev, rng, "f32", 2, 2, 48, 8, 4, [3, 9])
    k = rng.standard_normal((2, 2, 48)).astype(np.float32)
    v = rng.standard_normal((2, 2, 48)).astype(np.float32)
    hip_ctx.rope_append_device(c.handle, 1, dev.put(k), dev.put(v))
    hip_ctx.synchronize()
    keys, values = c.device("keys"), c.device("values")
    for s in range(2):
        p, o = c.at(s, int(c.lengths[s]))
        assert np.array_equal(keys[p, :, o], k[s]) and np.array_equal(values[p, :, o], v[s])


def test_append_reports_what_does_not_fit(hip_ctx, dev):
    rng = np.random.default_rng(2)
    rope, inv, mag = make_rope(dev, 32)
    for what in ("full", "page", "length"):
        c = R.Cache(dev, rng, "f16", 2, 2, 32, 8, 3, [22, 4])
        if what == "page":
            c.table[0, 2] = c.keys.shape[0]
            c.upload()
        if what == "length":
            c.lengths[0] = 0xFFFFFFF0
            c.upload()
        k = rng.standard_normal((2, 4, 2, 32)).astype(np.float32)
        hip_ctx.rope_append_device(c.handle, 4, dev.put(k), dev.put(k), rope=rope)
        with pytest.raises(HipError) as e:
            hip_ctx.synchronize()
        assert e.value.status == -9
        assert ("pool" if what == "page" else "do not fit") in e.value.message
        hip_ctx.synchronize()  # reported once
        values = c.device("values")
        want = c.values.copy()
        for s in range(2):
            for t in range(4):
                slot = int(c.lengths[s]) + t
                if slot < c.capacity and c.table[s, slot // 8] < c.keys.shape[0]:
                    p, o = c.at(s, slot)
                    want[p, :, o] = k[s, t].astype(np.float16)
        assert np.array_equal(values, want)


def test_advance(hip_ctx, dev):
    rng = np.random.default_rng(3)
    c = R.Cache(dev, rng, "f16", 300, 1, 8, 4, 3, rng.integers(0, 13, 300), spare=0)
    counts = rng.integers(0, 5, 300).astype(np.uint32)
    counts[7] = 0xFFFFFFFF
    hip_ctx.kv_advance_device(c.handle, dev.put(counts), 1)
    hip_ctx.synchronize()
    got = dev.get(c.d_lengths, c.lengths)
    want = np.minimum(c.lengths.astype(np.int64) + counts + 1, 12)
    assert np.array_equal(got, want)
    hip_ctx.kv_advance_device(c.handle, None, 2)
    hip_ctx.synchronize()
    assert np.array_equal(dev.get(c.d_lengths, c.lengths), np.minimum(want + 2, 12))


def test_rows_beyond_four_gigabytes(hip_ctx, dev):
    # pages at the end of a pool of more than 2^32 values
    kv, dim, page = 2, 256, 64
    pages = (1 << 32) // (kv * dim * page) + 70
    nbytes = pages * kv * dim * page * 2
    keys, values = dev.raw(nbytes), dev.raw(nbytes)
    table = np.array([[pages - 1, pages - 3]], np.uint32)
    h = si_hip.KvCache(ggml_type=30, kv_heads=kv, head_dim=dim, page_tokens=page, pages=pages,
                       sequences=1, max_pages=2, d_keys=keys, d_values=values,
                       d_page_table=dev.put(table), d_lengths=dev.put(np.array([62], np.uint32)))
    rng = np.random.default_rng(4)
    k = rng.standard_normal((4, kv, dim)).astype(np.float32)
    v = rng.standard_normal((4, kv, dim)).astype(np.float32)
    hip_ctx.rope_append_device(h, 4, dev.put(k), dev.put(v))
    hip_ctx.synchronize()
    for t in range(4):
        p, o = int(table[0, (62 + t) // page]), (62 + t) % page
        for head in range(kv):
            at = (((p * kv + head) * page) + o) * dim * 2
            assert np.array_equal(dev.ctx.from_device(keys + at, (dim,), np.uint16),
                                  R.to_bf16(k[t, head]))
            assert np.array_equal(dev.ctx.from_device(values + at, (dim,), np.uint16),
                                  R.to_bf16(v[t, head]))


def test_more_tokens_than_a_launch_has_threads_for(hip_ctx, dev):
    """2^24 tokens and some: a workgroup of 256 threads each is 2^32 threads."""
    n = (1 << 24) + 5
    rng = np.random.default_rng(6)
    rope, inv, mag = make_rope(dev, 2, 1e4)
    x = rng.standard_normal((n, 2)).astype(np.float32)
    pos = np.arange(n, dtype=np.uint32)
    d_x, d_p = dev.put(x), dev.put(pos)
    d_y = dev.put(np.full_like(x, 7.0))
    hip_ctx.rope_device(rope, d_x, n, 1, 2, d_p, d_y)
    hip_ctx.synchronize()
    want, size = R.rotate(x[:, None], pos, inv, mag, 0)
    # beyond 2^20 positions the f64 reference's angle is itself off by pos * 2^-53 radians
    check(dev.get(d_y, x)[:, None], want, size + 1e-8)

    page = 1 << 12
    pages = n // page + 1
    order = rng.permutation(pages).astype(np.uint32)
    d_keys, d_values = (dev.put(np.full((pages * page, 2), 3.0, np.float32)) for _ in range(2))
    h = si_hip.KvCache(ggml_type=0, kv_heads=1, head_dim=2, page_tokens=page, pages=pages,
                       sequences=1, max_pages=pages, d_keys=d_keys, d_values=d_values,
                       d_page_table=dev.put(order), d_lengths=dev.put(np.zeros(1, np.uint32)))
    hip_ctx.rope_append_device(h, n, d_x, d_x, rope=rope, d_q=d_x, heads=1, d_q_out=d_y)
    hip_ctx.synchronize()
    check(dev.get(d_y, x)[:, None], want, size + 1e-8, "query")
    slots = np.arange(n)
    row = order[slots // page].astype(np.int64) * page + slots % page
    like = np.empty((pages * page, 2), np.float32)
    assert np.array_equal(dev.get(d_values, like)[row], x)
    check(dev.get(d_keys, like)[row][:, None], want, size + 1e-8, "keys")
