"""GPU: eviction by accumulated weight, to the slot and bit."""
import numpy as np
import pytest

import decode_ref as R
from si_hip import HipError

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(hip_ctx):
    d = R.Device(hip_ctx)
    yield d
    hip_ctx.synchronize()
    d.free()


def evict(ctx, dev, c, weights, keep, sinks, recent, page=None, offset=0, one_pool=False):
    """Runs it and checks everything it wrote and everything it must not."""
    rng = np.random.default_rng(keep)
    b, kv = len(c.lengths), c.kv_heads
    to = R.Cache(dev, rng, c.kind, b, kv, c.head_dim, page or c.page, -(-keep // (page or c.page)),
                 [77] * b, offset)
    if one_pool:
        to.table = to.table + c.keys.shape[0]
        both = [np.concatenate([x, y]) for x, y in ((c.keys, to.keys), (c.values, to.values))]
        c.keys, c.values = to.keys, to.values = both
        c.upload()
        to.upload()
        to.handle.d_keys, to.handle.d_values = to.d_keys, to.d_values = c.d_keys, c.d_values
    tw = rng.random((b, kv, keep + 5)).astype(np.float32)
    kept = np.full((b, kv, keep), 123456, np.uint32)
    d_w, d_tw, d_kept = dev.put(weights), dev.put(tw), dev.put(kept)
    ctx.kv_evict_device(c.handle, d_w, weights.shape[2], keep, sinks, recent, to.handle, d_tw,
                        keep + 5, d_kept)
    ctx.synchronize()
    keys, values = to.keys.copy(), to.values.copy()
    for s in range(b):
        n = min(int(c.lengths[s]), c.capacity)
        for h in range(kv):
            slots = R.kept_slots(weights[s, h], n, keep, sinks, recent)
            assert len(slots) == min(n, keep)
            kept[s, h] = R.NONE
            kept[s, h, :len(slots)] = slots
            tw[s, h, :len(slots)] = weights[s, h, slots]
            for i, slot in enumerate(slots):
                (p, o), (tp, to_o) = c.at(s, slot), to.at(s, i)
                keys[tp, h, to_o], values[tp, h, to_o] = c.keys[p, h, o], c.values[p, h, o]
    assert np.array_equal(dev.get(d_kept, kept), kept)
    assert np.array_equal(dev.get(d_tw, tw).view(np.uint32), tw.view(np.uint32))
    assert np.array_equal(to.device("keys"), keys) and np.array_equal(to.device("values"), values)
    assert np.array_equal(dev.get(to.d_lengths, to.lengths), np.minimum(c.lengths, keep))
    assert np.array_equal(dev.get(c.d_lengths, c.lengths), c.lengths)
    assert np.array_equal(dev.get(d_w, weights).view(np.uint32), weights.view(np.uint32))


@pytest.mark.parametrize("kind,dim,page,offset", [("bf16", 256, 16, 0), ("f16", 128, 7, 0),
                                                  ("f32", 64, 32, 0), ("f16", 80, 5, 8),
                                                  ("bf16", 33, 16, 0), ("f32", 33, 3, 4),
                                                  ("f16", 1, 4, 2), ("bf16", 250, 16, 0),
                                                  ("f32", 256, 16, 0)])
@pytest.mark.parametrize("keep,sinks,recent", [(64, 4, 16), (1, 0, 0), (1, 1, 0), (20, 0, 20),
                                               (100, 40, 60), (127, 0, 1), (130, 3, 0)])
def test_heads_and_budgets(hip_ctx, dev, kind, dim, page, offset, keep, sinks, recent):
    rng = np.random.default_rng(dim + keep)
    lengths = [0, 1, 63, 64, 65, 130, 200]
    c = R.Cache(dev, rng, kind, 7, 2, dim, page, -(-200 // page), lengths, offset)
    w = rng.random((7, 2, c.capacity + 3)).astype(np.float32)
    evict(hip_ctx, dev, c, w, keep, sinks, recent, page=11, offset=offset)


@pytest.mark.parametrize("case", ["equal", "few values", "zeros", "signed zeros", "nan", "infinities",
                                  "near", "subnormal", "negative"])
def test_ties_and_strange_weights(hip_ctx, dev, case):
    rng = np.random.default_rng(len(case))
    c = R.Cache(dev, rng, "f16", 3, 2, 16, 16, 160, [2500, 1200, 1025])
    shape = (3, 2, c.capacity)
    w = {"equal": lambda: np.full(shape, 0.25),
         "few values": lambda: rng.integers(0, 4, shape) / 3,
         "zeros": lambda: np.where(rng.random(shape) < 0.9, 0.0, rng.random(shape)),
         "signed zeros": lambda: np.where(rng.random(shape) < 0.5, 0.0, -0.0),
         "nan": lambda: np.where(rng.random(shape) < 0.7, np.nan, rng.random(shape) - 0.5),
         "infinities": lambda: rng.choice([np.inf, -np.inf, 1.0, np.nan, 3e38, -3e38], shape),
         "near": lambda: (np.float32(1.0) + rng.integers(0, 9, shape) * 2.0 ** -23),
         "subnormal": lambda: rng.integers(0, 50, shape) * 1e-45,
         "negative": lambda: -rng.random(shape)}[case]().astype(np.float32)
    evict(hip_ctx, dev, c, w, 1000, 5, 50)
    evict(hip_ctx, dev, c, w, 1024, 0, 0)


@pytest.mark.parametrize("n,keep", [(1023, 512), (1024, 1000), (1025, 1024), (4095, 7), (4096, 4095),
                                    (9999, 5000), (70001, 33333)])
def test_long_rows(hip_ctx, dev, n, keep):
    rng = np.random.default_rng(n)
    c = R.Cache(dev, rng, "f16", 1, 3, 8, 64, -(-n // 64), [n])
    w = np.exp(rng.standard_normal((1, 3, c.capacity)) * 3).astype(np.float32)
    w[rng.random(w.shape) < 0.2] = 0.0
    evict(hip_ctx, dev, c, w, keep, 3, min(64, keep - 3))


def test_inside_one_pool(hip_ctx, dev):
    rng = np.random.default_rng(21)
    c = R.Cache(dev, rng, "bf16", 2, 2, 64, 16, 12, [190, 33])
    evict(hip_ctx, dev, c, rng.random((2, 2, c.capacity)).astype(np.float32), 90, 4, 20, one_pool=True)


def test_reports(hip_ctx, dev):
    rng = np.random.default_rng(22)
    for what in ("source", "destination", "length"):
        c = R.Cache(dev, rng, "f16", 1, 2, 32, 8, 8, [60])
        to = R.Cache(dev, rng, "f16", 1, 2, 32, 8, 4, [0])
        if what == "source":
            c.table[0, 0] = 1000
        elif what == "destination":
            to.table[0, 1] = 0xFFFFFFFF
        else:
            c.lengths[0] = 65
        c.upload()
        to.upload()
        w = rng.random((1, 2, 64)).astype(np.float32)
        d_kept = dev.put(np.zeros((1, 2, 30), np.uint32))
        d_tw = dev.put(np.zeros((1, 2, 32), np.float32))
        hip_ctx.kv_evict_device(c.handle, dev.put(w), 64, 30, 8, 4, to.handle, d_tw, 32, d_kept)
        with pytest.raises(HipError) as e:
            hip_ctx.synchronize()
        assert ("do not fit" if what == "length" else "pool") in e.value.message
        # all rows but those on the page that is not there
        values, want = to.device("values"), to.values.copy()
        for h in range(2):
            for i, slot in enumerate(R.kept_slots(w[0, h], min(int(c.lengths[0]), 64), 30, 8, 4)):
                (p, o), (tp, to_o) = c.at(0, slot), to.at(0, i)
                if p < c.keys.shape[0] and tp < to.keys.shape[0]:
                    want[tp, h, to_o] = c.values[p, h, o]
        assert np.array_equal(values, want)


def test_refuses_to_write_what_it_reads(hip_ctx, dev):
    rng = np.random.default_rng(23)
    c = R.Cache(dev, rng, "f16", 1, 1, 8, 8, 4, [30])
    w = dev.put(np.zeros((1, 1, 32), np.float32))
    with pytest.raises(HipError) as e:
        hip_ctx.kv_evict_device(c.handle, w, 32, 8, 0, 0, c.handle, w, 32, w)
    assert e.value.status == -7


@pytest.mark.parametrize("n,keep", [(16384, 9000), (16385, 9000), (30001, 20000), (32767, 1),
                                    (32768, 32767), (32769, 9)])
@pytest.mark.parametrize("ties", [False, True])
def test_rows_held_by_a_workgroup(hip_ctx, dev, n, keep, ties):
    """Around the capacities up to which a thread holds 16 or 32 slots."""
    rng = np.random.default_rng(n + ties)
    c = R.Cache(dev, rng, "bf16", 2, 2, 8, 32, -(-n // 32), [n, n // 2 + 1])
    w = np.exp(rng.standard_normal((2, 2, c.capacity)) * 3).astype(np.float32)
    if ties:
        w = np.round(np.log2(w)).astype(np.float32)
    w[rng.random(w.shape) < 0.1] = 0.0
    evict(hip_ctx, dev, c, w, keep, min(5, keep - 1), min(64, keep // 2), page=16)
