"""GPU: softmax of logits against 64 bits, and the verification of drafted
tokens against exact integer arithmetic.

Softmax tolerance, per value: (x - m) / T is rounded twice, which moves its
exponential by 2^-23 |x - m| / T; exp2, the sum (f32, of at most some hundred
thousand terms in trees of 16 and 64) and the division round by a few units
more: 2^-23 (|x - m| / T + 24).
"""
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


def softmax64(x, t):
    x = x.astype(np.float64)
    z = (x - x.max(1, keepdims=True)) / np.float64(np.float32(t))
    e = np.exp(z)
    y = e / e.sum(1, keepdims=True)
    return y, 2.0 ** -23 * (np.where(np.isfinite(z), np.abs(z), 0) + 24) * y + 2.0 ** -140


def softmax(ctx, dev, x, t, offset=0, in_place=False):
    d_x = dev.put(x, offset)
    d_y = d_x if in_place else dev.put(np.full_like(x, 3.0), offset)
    ctx.softmax_device(d_x, x.shape[0], x.shape[1], t, d_y)
    ctx.synchronize()
    return dev.get(d_y, x)


@pytest.mark.parametrize("cols", [1, 2, 3, 63, 64, 255, 1000, 4095, 4096, 4097, 8192, 16385, 50257,
                                  151936])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_softmax(hip_ctx, dev, rows, cols):
    if rows == 300 and cols > 5000:
        rows = 20
    rng = np.random.default_rng(cols + rows)
    x = (rng.standard_normal((rows, cols)) * 4).astype(np.float32)
    for t, offset, in_place in [(1.0, 0, False), (0.3, 4, False), (1.7, 0, True)]:
        want, tol = softmax64(x, t)
        err = np.abs(softmax(hip_ctx, dev, x, t, offset, in_place) - want)
        assert np.all(err <= tol), f"{np.max(err / tol):.3f}"


def test_softmax_many_rows(hip_ctx, dev):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((70001, 9)).astype(np.float32)
    want, tol = softmax64(x, 0.5)
    assert np.all(np.abs(softmax(hip_ctx, dev, x, 0.5) - want) <= tol)


def test_softmax_masks_and_extremes(hip_ctx, dev):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, 9001)).astype(np.float32)
    x[0, ::2] = -np.inf
    x[1, :9000] = -np.inf
    x[2, :] = np.finfo(np.float32).min
    x[3, 5:] = np.finfo(np.float32).min
    x[4] *= 1e30
    x[5] = 1e30
    x[6, 4096:8192] = -np.inf
    x[7, :4096] = -np.inf
    for t in (1.0, 0.01, 50.0):
        with np.errstate(over="ignore", invalid="ignore"):
            want, tol = softmax64(x, t)
        got = softmax(hip_ctx, dev, x, t)
        assert np.all(np.abs(got - want) <= tol), np.argwhere(~(np.abs(got - want) <= tol))[:4]
    # rows without a finite value, or with one that is no number, are none; the others are not touched
    x[0] = -np.inf
    x[1, 77] = np.nan
    x[3, 8000] = np.inf
    want, tol = softmax64(x[4:], 1.0)
    got = softmax(hip_ctx, dev, x, 1.0)
    assert np.isnan(got[0]).all() and np.isnan(got[1]).all() and np.isnan(got[3, 8000])
    assert np.all(np.abs(got[4:] - want) <= tol)


# ---- verification ------------------------------------------------------------------

def probabilities(rng, shape, sharp=2.0):
    e = np.exp(rng.standard_normal(shape) * sharp)
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def verify(ctx, dev, target, draft, tokens, counts, uniform, vocab):
    n, m = tokens.shape
    d_a, d_o = dev.put(np.full(n, 99, np.uint32)), dev.put(np.full((n, m + 1), 99, np.uint32))
    ctx.verify_draft_device(dev.put(target), None if draft is None else dev.put(draft),
                            dev.put(tokens), dev.put(uniform), n, m, vocab, d_a, d_o,
                            d_counts=None if counts is None else dev.put(counts))
    error = None
    try:
        ctx.synchronize()
    except HipError as e:
        error = e.message
    return dev.get(d_a, np.empty(n, np.uint32)), dev.get(d_o, np.empty((n, m + 1), np.uint32)), error


def check(ctx, dev, target, draft, tokens, counts, uniform, vocab):
    accepted, out, error = verify(ctx, dev, target, draft, tokens, counts, uniform, vocab)
    want_a, want_o = R.verify(target, draft, tokens, counts, uniform, vocab)
    assert np.array_equal(accepted, want_a)
    assert np.array_equal(out, want_o)
    return accepted, out, error


@pytest.mark.parametrize("vocab", [1, 2, 15, 16, 17, 255, 1000, 4096, 4097, 12289])
@pytest.mark.parametrize("drafts", [1, 3, 16])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(hip_ctx, dev, vocab, drafts, certain):
    rng = np.random.default_rng(vocab * 17 + drafts)
    n = 6
    target = probabilities(rng, (n, drafts + 1, vocab))
    draft = None if certain else probabilities(rng, (n, drafts, vocab), 1.0)
    if not certain:  # near enough to the target for drafts to be accepted
        draft = (0.9 * target[:, :drafts] + 0.1 * draft).astype(np.float32)
    tokens = np.argmax(target[:, :drafts] if certain else draft / -np.log(rng.random(draft.shape)),
                       2).astype(np.uint32)
    for uniform in (rng.random((n, drafts + 1)), np.zeros((n, drafts + 1)),
                    np.full((n, drafts + 1), 1 - 2.0 ** -24)):
        uniform = uniform.astype(np.float32)
        for counts in (None, rng.integers(0, drafts + 1, n).astype(np.uint32),
                       np.array([0, drafts, 0xFFFFFFFF, 0, 1, 1], np.uint32)):
            _, _, error = check(hip_ctx, dev, target, draft, tokens, counts, uniform, vocab)
            assert error is None


def test_verify_follows_the_target(hip_ctx, dev):
    """Over many sequences the first token is distributed as the target's row,
    whatever the drafter's: five sigma of a binomial."""
    rng = np.random.default_rng(5)
    n, vocab = 40000, 8
    p, q = probabilities(rng, (vocab,), 1.0), probabilities(rng, (vocab,), 1.0)
    target = np.broadcast_to(p, (n, 2, vocab)).copy()
    draft = np.broadcast_to(q, (n, 1, vocab)).copy()
    tokens = rng.choice(vocab, (n, 1), p=q.astype(np.float64) / q.sum(dtype=np.float64)).astype(np.uint32)
    uniform = rng.random((n, 2), np.float32)
    accepted, out, error = verify(hip_ctx, dev, target, draft, tokens, None, uniform, vocab)
    assert error is None and 0 < accepted.sum() < n
    share = np.bincount(out[:, 0], minlength=vocab) / n
    assert np.all(np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-4)


def test_verify_degenerate_rows(hip_ctx, dev):
    rng = np.random.default_rng(6)
    n, m, vocab = 7, 2, 5000
    target = probabilities(rng, (n, m + 1, vocab))
    draft = target[:, :m].copy()  # nothing is left of p - q: the token comes from p
    tokens = rng.integers(0, vocab, (n, m)).astype(np.uint32)
    uniform = rng.random((n, m + 1)).astype(np.float32)
    uniform[:, 0] = np.float32(1.0)  # refuses (outside [0, 1), still defined)
    target[1, :, ::3] = np.nan
    draft[2, :, ::5] = np.nan
    target[3, 0] = 0.0
    target[3, 0, 4999] = 1.0
    draft[3, 0] = 0.0
    target[4, 0, 17] = np.inf
    uniform[5] = np.nan
    uniform[6] = -1.0
    _, _, error = check(hip_ctx, dev, target, draft, tokens, None, uniform, vocab)
    assert error is None
    # sums that need more than 64 bits times 24: rows that do not add up to 1
    big = rng.random((n, m + 1, vocab)).astype(np.float32) * 0.5 + 0.5
    _, _, error = check(hip_ctx, dev, big, None, tokens, np.zeros(n, np.uint32), uniform, vocab)
    assert error is None


def test_verify_reports(hip_ctx, dev):
    rng = np.random.default_rng(7)
    vocab = 300
    target = probabilities(rng, (3, 3, vocab))
    draft = probabilities(rng, (3, 2, vocab))
    tokens = np.array([[1, 2], [vocab, 3], [4, 5]], np.uint32)
    uniform = np.full((3, 3), 0.5, np.float32)
    uniform[2, 0] = 1.0
    for q in (draft, None):
        _, _, error = check(hip_ctx, dev, target, q, tokens, None, uniform, vocab)
        assert "beyond the vocabulary" in error
        # behind the first refused one it is not looked at
        later = np.array([[1, 2], [2, 3], [4, 0xFFFFFFFF]], np.uint32)
        t = target.copy()
        t[2, 0, 4] = 0.0
        _, _, error = check(hip_ctx, dev, t, q, later, None, uniform, vocab)
        assert error is None
    target[1] = 0.0
    target[2] = np.nan
    tokens[1, 0] = 0
    accepted, out, error = check(hip_ctx, dev, target, draft, tokens, None, uniform, vocab)
    assert "zero throughout" in error
    assert out[1, 0] == R.NONE and out[2, 0] == R.NONE


def test_verify_many_sequences(hip_ctx, dev):
    rng = np.random.default_rng(8)
    n, m, vocab = 700, 4, 33
    target, draft = probabilities(rng, (n, m + 1, vocab)), probabilities(rng, (n, m, vocab), 1.5)
    tokens = rng.integers(0, vocab, (n, m)).astype(np.uint32)
    check(hip_ctx, dev, target, draft, tokens, None, rng.random((n, m + 1)).astype(np.float32), vocab)


def test_verify_in_a_graph(hip_ctx, dev):
    """Logits to probabilities to tokens, replayed with other logits each time."""
    rng = np.random.default_rng(9)
    n, m, vocab = 2, 3, 5001
    logits = (rng.standard_normal((n * (m + 1), vocab)) * 3).astype(np.float32)
    tokens = rng.integers(0, vocab, (n, m)).astype(np.uint32)
    uniform = rng.random((n, m + 1)).astype(np.float32)
    d_x, d_p, d_u = dev.put(logits), dev.put(np.zeros_like(logits)), dev.put(uniform)
    d_t, d_a, d_o = dev.put(tokens), dev.put(np.zeros(n, np.uint32)), dev.put(np.zeros((n, m + 1), np.uint32))
    hip_ctx.capture_begin()
    hip_ctx.softmax_device(d_x, n * (m + 1), vocab, 0.8, d_p)
    hip_ctx.verify_draft_device(d_p, None, d_t, d_u, n, m, vocab, d_a, d_o)
    graph = hip_ctx.capture_end()
    for step in range(4):
        logits = (rng.standard_normal(logits.shape) * 3).astype(np.float32)
        tokens = logits.reshape(n, m + 1, vocab)[:, :m].argmax(2).astype(np.uint32)
        hip_ctx.to_device(d_x, logits)
        hip_ctx.to_device(d_t, tokens)
        graph.launch()
        hip_ctx.synchronize()
        p = dev.get(d_p, logits)
        want, tol = softmax64(logits, 0.8)
        assert np.all(np.abs(p - want) <= tol)
        want_a, want_o = R.verify(p.reshape(n, m + 1, vocab), None, tokens, None, uniform, vocab)
        assert np.array_equal(dev.get(d_a, np.empty(n, np.uint32)), want_a)
        assert np.array_equal(dev.get(d_o, np.empty((n, m + 1), np.uint32)), want_o)


def test_draw_in_steps_of_a_uniform_number(hip_ctx, dev):
    """The number that draws is taken down to a multiple of 2^-24: below that the first token with
    any mass is drawn, though the numbers themselves lie beyond it."""
    vocab = 6000
    target = np.zeros((6, 2, vocab), np.float32)
    target[:, :, 17] = 2.0 ** -30
    target[:, :, 4100] = 2.0 ** -24
    target[:, :, 5000] = 1.0 - 2.0 ** -23
    tokens = np.zeros((6, 1), np.uint32)
    uniform = np.zeros((6, 2), np.float32)
    uniform[:, 1] = [0.0, 2.0 ** -29, 2.0 ** -24 - 2.0 ** -48, 2.0 ** -24, 1.5 * 2.0 ** -24, 2.0 ** -23]
    accepted, out, error = check(hip_ctx, dev, target, None, tokens, np.zeros(6, np.uint32), uniform,
                                 vocab)
    assert error is None and not accepted.any()
    assert out[:, 0].tolist() == [17, 17, 17, 4100, 4100, 5000]


def test_verify_a_vocabulary_of_many_chunks(hip_ctx, dev):
    """More chunks of 4096 than a workgroup has threads: each looks for the draw in two."""
    rng = np.random.default_rng(10)
    n, m, vocab = 4, 1, (256 + 20) * 4096 + 11
    target = probabilities(rng, (n, m + 1, vocab), 1.0)
    draft = probabilities(rng, (n, m, vocab), 1.0)
    target[2, :, :vocab - 5] = 0.0
    tokens = rng.integers(0, vocab, (n, m)).astype(np.uint32)
    uniform = np.array([[0.999, 0.3], [0.999, 0.97], [1.0, 0.6], [0.0, 1 - 2.0 ** -24]], np.float32)
    for q in (draft, None):
        _, out, error = check(hip_ctx, dev, target, q, tokens, None, uniform, vocab)
        assert error is None and out[2, 0] >= vocab - 5
