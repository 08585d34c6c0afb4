"""GPU: head norms, positions of several axes and the cache append against 64 bits.

Tolerance of a value: its pair's |a| + |b| after the norm, times 2e-6.  The sum of up to 256 squares
is added up in at most 38 roundings, all of one sign, and halved by the root: 19 U = 1.1e-6 (U = 2^-24);
its quotient, eps, root, reciprocal and two or three products 6 U = 3.6e-7; the rotation as
without a norm 5e-7 (test_gpu_rope).
"""
import numpy as np
import pytest

import decode_ref as R
import mixer_ref as M
import si_hip
from si_hip import HipError

pytestmark = pytest.mark.gpu
REL = 2e-6
NAN = np.float32(np.nan)


@pytest.fixture
def dev(hip_ctx):
    d = R.Device(hip_ctx)
    yield d
    hip_ctx.synchronize()
    d.free()


class Call:
    """A norm, a rotation and its axes over some rows, each of which may be missing."""

    def __init__(self, dev, rng, rows, dim, n, layout=0, sections=None, order=0, norm="plain", theta=1e6):
        self.weights = [None, None]
        self.norm = self.rope = self.axes = self.positions = self.d_positions = self.table = None
        self.layout, self.plus_one = layout, int(norm == "plus_one")
        if norm:
            if norm != "ones":
                self.weights = [rng.standard_normal(dim).astype(np.float32) for _ in range(2)]
            self.norm = si_hip.HeadNorm(
                eps=1e-6, plus_one=self.plus_one,
                d_q_weight=None if norm == "ones" else dev.put(self.weights[0]),
                d_k_weight=None if norm == "ones" else dev.put(self.weights[1]))
            if norm == "ones":
                self.weights = [1.0, 1.0]
        if n:
            self.table, magnitude = si_hip.rope_frequencies(n, theta)
            self.rope = si_hip.Rope(layout=layout, rotary_dim=n, magnitude=magnitude,
                                    d_frequencies=dev.put(self.table))
            count = len(sections) if sections else 1
            pos = rng.integers(0, 1 << 18, (count, rows)).astype(np.uint32)
            pos[:, 0] = (1 << 32) - 1
            self.axis = np.zeros(n // 2, np.uint8)
            if sections:
                self.axis = si_hip.rope_axis_table(n, sections, order)
                self.axes = si_hip.RopeAxes(axes=count, d_axis=dev.put(self.axis))
            self.set(dev, pos)

    def set(self, dev, pos):
        self.d_positions = dev.put(pos)
        self.positions = pos[self.axis].T  # [rows][pairs]

    def want(self, x, which):
        return M.norm_rope(x, self.weights[which] if self.norm else None,
                           np.float64(np.float32(1e-6)), self.plus_one, self.table, self.positions,
                           self.layout)


def check(got, want, size, what=""):
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= REL * size + 1e-30), f"{what}: {np.max(err / (REL * size + 1e-30)):.3f}"


SHAPES = [(128, 128, None, 0), (256, 64, [11, 11, 10], 1), (64, 64, [5, 20, 7], 0), (80, 40, [10, 10], 0),
          (96, 2, None, 0), (33, 10, [2, 1, 1, 1], 1), (2, 2, [1], 0), (128, 12, [0, 6], 0), (256, 256, None, 0),
          (255, 254, [100, 27], 0), (72, 0, None, 0), (1, 0, None, 0), (256, 0, None, 0)]


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("norm", ["plain", "plus_one", "ones", None])
@pytest.mark.parametrize("dim,n,sections,order", SHAPES)
def test_rows(hip_ctx, dev, dim, n, sections, order, norm, layout):
    if not n and (norm is None or layout):
        pytest.skip("nothing to do, or no layout")
    rng = np.random.default_rng(dim * 7 + n + layout)
    for tokens, heads, pad, offset in [(1, 1, 0, 0), (5, 3, 0, 0), (37, 7, 4, 0), (3, 50, 1, 4)]:
        c = Call(dev, rng, tokens, dim, n, layout, sections, order, norm)
        x = (rng.standard_normal((tokens, heads, dim + pad)) * 3).astype(np.float32)
        want, size = c.want(x[..., :dim], 0)
        d_x = dev.put(x, offset)
        d_y = dev.put(np.full((tokens, heads, dim), 7.0, np.float32), offset)
        args = dict(norm=c.norm, rope=c.rope, axes=c.axes, d_positions=c.d_positions)
        hip_ctx.norm_rope_device(d_x, tokens, heads, dim, d_y, head_stride=dim + pad, **args)
        hip_ctx.synchronize()
        check(dev.get(d_y, want.astype(np.float32)), want, size, f"{tokens}x{heads}")
        hip_ctx.norm_rope_device(d_x, tokens, heads, dim, d_x, head_stride=dim + pad,
                                 y_head_stride=dim + pad, **args)
        hip_ctx.synchronize()
        got = dev.get(d_x, x)
        check(got[..., :dim], want, size, "in place")
        assert np.array_equal(got[..., dim:], x[..., dim:])  # what lies between rows


def test_many_rows(hip_ctx, dev):
    """More tokens than one workgroup's, one head: several tokens a workgroup."""
    rng = np.random.default_rng(3)
    for tokens, heads, dim in [(8195, 1, 64), (2051, 5, 20), (1025, 30, 128)]:
        c = Call(dev, rng, tokens, dim, 16, 1, [3, 3, 2], 1, "plus_one")
        x = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
        want, size = c.want(x, 0)
        d_x = dev.put(x)
        hip_ctx.norm_rope_device(d_x, tokens, heads, dim, d_x, norm=c.norm, rope=c.rope, axes=c.axes,
                                 d_positions=c.d_positions)
        hip_ctx.synchronize()
        check(dev.get(d_x, x), want, size)


def test_numbers_that_are_none(hip_ctx, dev):
    """A head's NaN or infinity stays in that head; a head of zeros stays zero."""
    rng = np.random.default_rng(4)
    c = Call(dev, rng, 3, 64, 32, 0, None, 0, "plain")
    x = rng.standard_normal((3, 4, 64)).astype(np.float32)
    x[0, 1, 5], x[1, 2, 60], x[2, 0] = NAN, np.inf, 0.0
    want, size = c.want(x, 0)
    d_x = dev.put(x)
    hip_ctx.norm_rope_device(d_x, 3, 4, 64, d_x, norm=c.norm, rope=c.rope, d_positions=c.d_positions)
    hip_ctx.synchronize()
    got = dev.get(d_x, x)
    bad = np.zeros((3, 4), bool)
    bad[0, 1] = bad[1, 2] = True
    assert np.all(np.isnan(got[0, 1])) and np.isnan(got[1, 2]).any()
    check(got[~bad], want[~bad], size[~bad])
    assert np.all(got[2, 0] == 0.0)


def step(kind):
    return {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,dim,kv,n,sections,order,norm,offset", [
    (16, 128, 4, 128, None, 0, "plain", 0), (7, 64, 2, 64, [12, 10, 10], 1, "plus_one", 0),
    (1, 80, 3, 40, [10, 10], 0, "ones", 0), (24, 33, 2, 32, None, 0, "plus_one", 0),
    (16, 256, 1, 64, [11, 11, 10], 1, "plus_one", 8), (5, 10, 2, 0, None, 0, "plain", 0),
    (8, 96, 2, 96, [16, 16, 16], 0, None, 0)])
def test_append(hip_ctx, dev, kind, page, dim, kv, n, sections, order, norm, offset):
    rng = np.random.default_rng(page * 131 + dim)
    for tokens, positions, counts in [(1, True, False), (5, False, True), (3 * page + 2, True, True)]:
        max_pages = -(-(tokens + 40) // page)
        lengths = [0, 17, max_pages * page - tokens]
        c = R.Cache(dev, rng, kind, 3, kv, dim, page, max_pages, lengths, offset)
        call = Call(dev, rng, 3 * tokens, dim, n, 0, sections, order, norm, 1e4)
        heads, gap = 2 * kv, 3
        k = (rng.standard_normal((3 * tokens, kv * dim + gap)) * 4).astype(np.float32)
        v = rng.standard_normal((3 * tokens, kv * dim + gap)).astype(np.float32)
        q = rng.standard_normal((3 * tokens, heads, 2 * dim)).astype(np.float32)
        num = np.array([tokens, 0, tokens - 1], np.uint32) if counts else None
        if n and not positions:
            slots = (np.asarray(lengths)[:, None] + np.arange(tokens)).reshape(-1)
            call.set(dev, np.tile(slots.astype(np.uint32), (len(sections or [0]), 1)))
            call.d_positions = None
        if num is not None:  # rows behind a sequence's are not read
            behind = np.arange(tokens)[None] >= num[:, None]
            for x in (k, v, q):
                x[behind.reshape(-1)] = NAN
        with np.errstate(invalid="ignore"):
            qw, qs = call.want(q[..., :dim], 0)
            kw, ks = call.want(k[:, :kv * dim].reshape(-1, kv, dim), 1)
        d_qo = dev.put(np.full((3 * tokens, heads, dim), 5.0, np.float32))
        hip_ctx.norm_rope_append_device(
            c.handle, tokens, dev.put(k), dev.put(v), norm=call.norm, rope=call.rope, axes=call.axes,
            d_counts=None if num is None else dev.put(num), d_positions=call.d_positions,
            k_token_stride=kv * dim + gap, v_token_stride=kv * dim + gap, d_q=dev.put(q),
            heads=heads, q_head_stride=2 * dim, d_q_out=d_qo)
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
                err = np.abs(R.decode(keys[p, :, o], kind) - kw[row])
                assert np.all(err <= REL * ks[row] + step(kind) * np.abs(kw[row]) + 2.0 ** -24)
                assert np.array_equal(values[p, :, o],
                                      R.encode(v[row, :kv * dim].reshape(kv, dim), kind))
                check(q_out[row], qw[row], qs[row], "query")
                wk[p, :, o], wv[p, :, o] = keys[p, :, o], values[p, :, o]
        # every other row of the pool is as it was
        assert np.array_equal(keys, wk) and np.array_equal(values, wv)
        assert np.array_equal(dev.get(c.d_lengths, c.lengths), c.lengths)


def test_append_alone_is_the_plain_append(hip_ctx, dev):
    """Without a norm, one axis: what rope_append_device stores, bit by bit; without anything, the rows."""
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((6, 2, 64)).astype(np.float32) for _ in range(2))
    got = []
    for which in range(3):
        c = R.Cache(dev, np.random.default_rng(6), "f32", 2, 2, 64, 8, 4, [3, 9])
        call = Call(dev, np.random.default_rng(7), 6, 64, 32, 0, None, 0, None)
        if which == 0:
            hip_ctx.rope_append_device(c.handle, 3, dev.put(k), dev.put(v), rope=call.rope,
                                       d_positions=call.d_positions)
        elif which == 1:
            hip_ctx.norm_rope_append_device(c.handle, 3, dev.put(k), dev.put(v), rope=call.rope,
                                            d_positions=call.d_positions)
        else:
            hip_ctx.norm_rope_append_device(c.handle, 3, dev.put(k), dev.put(v))
        hip_ctx.synchronize()
        got.append((c.device("keys"), c.device("values")))
    assert all(np.array_equal(a, b) for a, b in zip(got[0], got[1]))
    for s in range(2):
        for t in range(3):
            p, o = c.at(s, int(c.lengths[s]) + t)
            assert np.array_equal(got[2][0][p, :, o], k[s * 3 + t])
            assert np.array_equal(got[2][1][p, :, o], v[s * 3 + t])


def test_reports(hip_ctx, dev):
    """Tokens that do not fit, pages beyond the pool, and axes beyond the positions'."""
    rng = np.random.default_rng(2)
    for what in ("full", "page", "length", "axis"):
        c = R.Cache(dev, rng, "f16", 2, 2, 32, 8, 3, [22 if what != "axis" else 2, 4])
        if what == "page":
            c.table[0, 2] = c.keys.shape[0]
            c.upload()
        if what == "length":
            c.lengths[0] = 0xFFFFFFF0
            c.upload()
        call = Call(dev, rng, 8, 32, 32, 0, [8, 8], 0, "plain")
        if what == "axis":
            bad = call.axis.copy()
            bad[9] = 2
            call.axes = si_hip.RopeAxes(axes=2, d_axis=dev.put(bad))
        k = rng.standard_normal((2, 4, 2, 32)).astype(np.float32)
        hip_ctx.norm_rope_append_device(c.handle, 4, dev.put(k), dev.put(k), norm=call.norm,
                                        rope=call.rope, axes=call.axes, d_positions=call.d_positions)
        with pytest.raises(HipError) as e:
            hip_ctx.synchronize()
        assert e.value.status == -9
        keys = c.device("keys")
        wk, _ = call.want(k.reshape(8, 2, 32), 1)
        for t in range(4):  # the other sequence's rows are there
            p, o = c.at(1, 4 + t)
            rows = np.arange(16) != 9 if what == "axis" else np.arange(16) >= 0
            rows = np.concatenate([rows, rows])
            assert np.allclose(R.decode(keys[p, :, o], "f16")[:, rows], wk[4 + t][:, rows], rtol=2e-3,
                               atol=2e-3)
    hip_ctx.synchronize()


def test_rows_beside_one_another(hip_ctx, dev):
    """Heads beside the gates of their outputs, normed into the gates' places and into a buffer that ends
    where theirs begins."""
    rng = np.random.default_rng(8)
    tokens, heads, dim = 9, 5, 64
    c = Call(dev, rng, tokens, dim, 32, 0, [6, 10], 0, "plain")
    x = rng.standard_normal((tokens, heads, 2, dim)).astype(np.float32)
    want, size = c.want(x[:, :, 0], 0)
    space = np.concatenate([np.zeros(tokens * heads * dim, np.float32), x.reshape(-1)])
    d = dev.put(space)
    d_x = d + 4 * tokens * heads * dim
    args = dict(norm=c.norm, rope=c.rope, axes=c.axes, d_positions=c.d_positions, head_stride=2 * dim)
    hip_ctx.norm_rope_device(d_x, tokens, heads, dim, d, **args)
    hip_ctx.norm_rope_device(d_x, tokens, heads, dim, d_x + 4 * dim, y_head_stride=2 * dim, **args)
    hip_ctx.synchronize()
    got = dev.get(d, space)
    check(got[:tokens * heads * dim].reshape(want.shape), want, size)
    got = got[tokens * heads * dim:].reshape(x.shape)
    check(got[:, :, 1], want, size)
    assert np.array_equal(got[:, :, 0], x[:, :, 0])


def test_one_axis_has_a_table(hip_ctx, dev):
    """A table for one axis is read like any other: zeros are axis 0, an entry beyond it is reported."""
    rng = np.random.default_rng(9)
    c = Call(dev, rng, 3, 64, 32, 0, [16], 0, "plain")
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    want, size = c.want(x, 0)
    args = dict(norm=c.norm, rope=c.rope, d_positions=c.d_positions)
    d_x, d_y = dev.put(x), dev.put(x)
    hip_ctx.norm_rope_device(d_x, 3, 2, 64, d_y, axes=c.axes, **args)
    hip_ctx.synchronize()
    check(dev.get(d_y, x), want, size)
    table = c.axis.copy()
    table[3] = 1
    bad = si_hip.RopeAxes(axes=1, d_axis=dev.put(table))
    hip_ctx.norm_rope_device(d_x, 3, 2, 64, d_y, axes=bad, **args)
    with pytest.raises(HipError) as e:
        hip_ctx.synchronize()
    assert e.value.status == -9
    check(dev.get(d_y, x), want, size)
