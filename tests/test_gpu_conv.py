"""GPU: the causal convolution against 64 bits (tolerance: mixer_ref.conv); states are exact."""
import numpy as np
import pytest

import decode_ref as R
import mixer_ref as M
import si_hip

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(hip_ctx):
    d = R.Device(hip_ctx)
    yield d
    hip_ctx.synchronize()
    d.free()


def check(got, want, tol):
    there = ~np.isnan(want)
    err = np.abs(got.astype(np.float64) - want)[there]
    assert np.all(err <= tol[there]), np.max(err / tol[there])
    assert np.all(got[~there] == 9.0)  # rows that are none of a sequence's stay as they were


def inputs(rng, n, tokens, channels, width, bias, fresh):
    x = rng.standard_normal((n, tokens, channels)).astype(np.float32)
    w = rng.standard_normal((channels, width)).astype(np.float32)
    b = rng.standard_normal(channels).astype(np.float32) if bias else None
    s = None if fresh else rng.standard_normal((n, width - 1, channels)).astype(np.float32)
    return x, w, b, s


@pytest.mark.parametrize("width", range(2, 9))
@pytest.mark.parametrize("n,tokens,channels,ragged,bias,act,fresh,offset", [
    (1, 1, 64, False, False, 1, False, 0), (3, 1, 33, False, True, 1, True, 4),
    (2, 2, 1, False, True, 0, False, 0), (4, 5, 258, True, False, 1, False, 0),
    (3, 9, 40, True, True, 1, True, 4), (2, 77, 131, True, True, 1, False, 8),
    (1, 300, 20, False, False, 0, False, 0)])
def test_conv(hip_ctx, dev, width, n, tokens, channels, ragged, bias, act, fresh, offset):
    rng = np.random.default_rng(width * 1000 + tokens)
    x, w, b, state = inputs(rng, n, tokens, channels, width, bias, fresh)
    counts = [tokens] * n
    if ragged:
        counts = [tokens, 0, max(tokens - 3, 1), 1][:n]
    for s in range(n):
        x[s, counts[s]:] = np.nan
    want, tol, states = M.conv(x, w, b, state, counts, act)
    opt = lambda a: None if a is None else dev.put(a, offset)  # noqa: E731
    d_counts = dev.put(np.array(counts, np.uint32)) if ragged else None
    for in_place in (False, True):
        d_state = opt(state)
        d_out = d_state if in_place and state is not None else dev.put(
            np.full((n, width - 1, channels), 3.0, np.float32), offset)
        d_y = dev.put(np.full(x.shape, 9.0, np.float32), offset)
        hip_ctx.causal_conv_device(dev.put(x, offset), opt(w), n, tokens, channels, width, d_y=d_y,
                                   d_bias=opt(b), activation=act, d_state=d_state, d_state_out=d_out,
                                   d_counts=d_counts)
        hip_ctx.synchronize()
        check(dev.get(d_y, x), want, tol)
        assert np.array_equal(dev.get(d_out, states), states)


def test_strides_and_parts(hip_ctx, dev):
    """Rows a stride apart; outputs alone; the state alone, `more` tokens further than counted."""
    rng = np.random.default_rng(1)
    n, tokens, channels, width = 3, 6, 70, 4
    x, w, b, state = inputs(rng, n, tokens, channels, width, True, False)
    wide = np.full((n, tokens, channels + 5), 4.0, np.float32)
    wide[..., :channels] = x
    d_x, d_w, d_b, d_state = dev.put(wide), dev.put(w), dev.put(b), dev.put(state)
    want, tol, states = M.conv(x, w, b, state, [tokens] * n, 1)
    out = np.full((n, tokens, channels + 3), 9.0, np.float32)
    d_y = dev.put(out)
    hip_ctx.causal_conv_device(d_x, d_w, n, tokens, channels, width, d_y=d_y, d_bias=d_b, d_state=d_state,
                               x_token_stride=channels + 5, y_token_stride=channels + 3)
    hip_ctx.synchronize()
    got = dev.get(d_y, out)
    check(got[..., :channels], want, tol)
    assert np.all(got[..., channels:] == 9.0)
    assert np.array_equal(dev.get(d_state, state), state)
    counts = np.array([0, 2, 0xFFFFFFFF], np.uint32)
    _, _, states = M.conv(x, w, b, state, [1, 3, tokens], 1)
    hip_ctx.causal_conv_device(d_x, d_w, n, tokens, channels, width, d_bias=d_b, d_state=d_state,
                               d_state_out=d_state, d_counts=dev.put(counts), more=1,
                               x_token_stride=channels + 5)
    hip_ctx.synchronize()
    assert np.array_equal(dev.get(d_state, state), states)


def test_token_by_token(hip_ctx, dev):
    """Runs of any length from the state of the one before: the same outputs, bit by bit."""
    rng = np.random.default_rng(2)
    channels, width, tokens = 36, 4, 40
    x, w, b, _ = inputs(rng, 1, tokens, channels, width, True, True)
    d_w, d_b, d_x = dev.put(w), dev.put(b), dev.put(x)
    whole = dev.put(np.zeros_like(x))
    hip_ctx.causal_conv_device(d_x, d_w, 1, tokens, channels, width, d_y=whole, d_bias=d_b)
    parts, d_state = dev.put(np.zeros_like(x)), dev.put(np.full((3, channels), 7.0, np.float32))
    t = 0
    for run in (1, 1, 2, 7, 1, 20, 8):
        hip_ctx.causal_conv_device(d_x + 4 * t * channels, d_w, 1, run, channels, width,
                                   d_y=parts + 4 * t * channels, d_bias=d_b,
                                   d_state=d_state if t else None, d_state_out=d_state)
        t += run
    hip_ctx.synchronize()
    assert t == tokens and np.array_equal(dev.get(whole, x), dev.get(parts, x))
    assert np.array_equal(dev.get(d_state, x[0, -3:]), x[0, -3:])


def test_numbers_that_are_none(hip_ctx, dev):
    """A NaN reaches its channel's outputs of its own and the next width - 1 tokens; large sums do not
    overflow in the activation."""
    rng = np.random.default_rng(3)
    x, w, _, state = inputs(rng, 1, 30, 12, 4, False, False)
    x[0, 7, 3], x[0, 25, 9] = np.nan, np.inf
    x[0, 12, 5], x[0, 13, 6] = 3e4, -3e4
    d_y = dev.put(np.full(x.shape, 9.0, np.float32))
    hip_ctx.causal_conv_device(dev.put(x), dev.put(w), 1, 30, 12, 4, d_y=d_y, d_state=dev.put(state))
    hip_ctx.synchronize()
    got = dev.get(d_y, x)
    bad = np.zeros(x.shape, bool)
    bad[0, 7:11, 3] = bad[0, 25:29, 9] = True
    clean = np.where(np.isfinite(x), x, 0).astype(np.float32)
    want, tol, _ = M.conv(clean, w, None, state, [30], 1)
    check(got[~bad], want[~bad], tol[~bad])
    assert np.all(np.isnan(got[0, 7:11, 3]))


@pytest.mark.parametrize("channels", [1, 4])
def test_more_runs_than_a_launch_has(hip_ctx, dev, channels):
    """Over 65535 runs of 64 tokens."""
    tokens, width = 65535 * 64 + 129, 2
    rng = np.random.default_rng(5)
    x, w, _, state = inputs(rng, 1, tokens, channels, width, False, False)
    d_y, d_out = dev.put(np.full(x.shape, 9.0, np.float32)), dev.put(np.zeros_like(state))
    hip_ctx.causal_conv_device(dev.put(x), dev.put(w), 1, tokens, channels, width, d_y=d_y,
                               activation=si_hip.CONV_NONE, d_state=dev.put(state), d_state_out=d_out)
    hip_ctx.synchronize()
    before = np.concatenate([state[0], x[0, :-1]])
    want = x[0].astype(np.float64) * w[:, 1] + before.astype(np.float64) * w[:, 0]
    size = np.abs(x[0] * w[:, 1]) + np.abs(before * w[:, 0])
    # (three roundings of at most half a step: two products and their sum)
    assert np.all(np.abs(dev.get(d_y, x)[0] - want) <= 1.1 * 3 * M.U * size + 1e-36)
    assert np.array_equal(dev.get(d_out, state)[0], x[0, -1:])


def test_rows_beside_one_another(hip_ctx, dev):
    """Inputs and outputs in the same rows of one buffer, each between the other's."""
    rng = np.random.default_rng(6)
    n, tokens, channels, width = 2, 70, 40, 4
    x, w, b, state = inputs(rng, n, tokens, channels, width, True, False)
    rows = np.full((n, tokens, 2 * channels + 3), 9.0, np.float32)
    rows[..., channels + 2:2 * channels + 2] = x
    want, tol, states = M.conv(x, w, b, state, [tokens] * n, 1)
    d, d_state = dev.put(rows), dev.put(state)
    hip_ctx.causal_conv_device(d + 4 * (channels + 2), dev.put(w), n, tokens, channels, width, d_y=d + 4,
                               d_bias=dev.put(b), d_state=d_state, d_state_out=d_state,
                               x_token_stride=2 * channels + 3, y_token_stride=2 * channels + 3)
    hip_ctx.synchronize()
    got = dev.get(d, rows)
    check(got[..., 1:channels + 1], want, tol)
    got[..., 1:channels + 1] = 9.0
    assert np.array_equal(got, rows) and np.array_equal(dev.get(d_state, states), states)


def test_activation(hip_ctx, dev):
    """SiLU of values from 9 to 17, where e^-y is below 2^-12 and its own error below 2^-11 U of the sum: the sum and
    the quotient round to half a step, U each, and what corrects the quotient adds less than 2^-20 U. And of any
    finite value, with the exponential's error of up to 2 U."""
    rng = np.random.default_rng(10)
    channels = 1 << 16
    w = np.zeros((channels, 2), np.float32)
    w[:, 1] = 1.0
    for low, high, tol in [(9.0, 17.0, 2.001 * M.U), (-80.0, 9.0, 4.001 * M.U), (-3.4e38, 3.4e38, 2.001 * M.U)]:
        y = rng.uniform(low, high, (1, channels)).astype(np.float32)
        d_out = dev.put(np.zeros_like(y))
        hip_ctx.causal_conv_device(dev.put(y), dev.put(w), 1, 1, channels, 2, d_y=d_out)
        hip_ctx.synchronize()
        want = M.silu(y.astype(np.float64))
        err = np.abs(dev.get(d_out, y) - want)
        assert np.all(err <= tol * np.abs(want) + 1e-36), np.max(err / (np.abs(want) + 1e-36)) / M.U
