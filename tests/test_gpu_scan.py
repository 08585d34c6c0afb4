"""GPU: the state scan against 64 bits (tolerances: mixer_ref.Scan)."""
import copy

import numpy as np
import pytest

import decode_ref as R
import mixer_ref as M
import si_hip

pytestmark = pytest.mark.gpu
DELTA, SELECTIVE = si_hip.SCAN_DELTA, si_hip.SCAN_SELECTIVE


@pytest.fixture
def dev(hip_ctx):
    d = R.Device(hip_ctx)
    yield d
    hip_ctx.synchronize()
    d.free()


def outputs(dev, scan, fill=9.0):
    n, tokens, _, vh, dk, dv = scan.shape
    return np.full((n, tokens, vh, dv), fill, np.float32), np.full((n, vh, dk, dv), fill, np.float32)


def within(got, want, tol, what=""):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {np.nanmax(err / tol):.3f} of the tolerance, {bad.sum()} values, first {np.argwhere(bad)[0]}"


def check_out(got, want, tol):
    there = ~np.isnan(want)
    within(got[there], want[there], tol[there], "out")
    assert np.all(got[~there] == 9.0)  # rows that are none of a sequence's stay as they were


def run(ctx, dev, scan, in_place=True):
    """Outputs and new states of one call."""
    scan.put(dev)
    out, state = outputs(dev, scan)
    d_out = dev.put(out)
    d_state_out = scan.d_state if in_place and scan.state is not None else dev.put(state)
    scan.call(ctx, scan.d_state, d_state_out, d_out)
    ctx.synchronize()
    return dev.get(d_out, out), dev.get(d_state_out, state)


SHAPES = [(2, 4, 128, 128), (1, 3, 64, 64), (2, 2, 128, 64), (1, 2, 96, 160), (1, 2, 192, 256),
          (2, 4, 40, 72), (3, 3, 16, 80), (1, 2, 1, 1), (1, 1, 7, 5), (1, 2, 33, 31), (1, 1, 256, 130),
          (2, 2, 127, 129)]


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("tokens", [1, 2, 5, 16, 17, 31, 32, 33, 64, 97])
@pytest.mark.parametrize("kh,vh,dk,dv", SHAPES)
def test_scan(hip_ctx, dev, kh, vh, dk, dv, tokens, rule):
    rng = np.random.default_rng(dk * 1009 + dv * 31 + tokens)
    order = (dk + tokens) % 2
    ragged = tokens % 2 == 1 and tokens > 1
    counts = [tokens, tokens // 2, 0] if ragged else None
    scan = M.Scan(rng, 3 if ragged else 1 + tokens % 3, tokens, kh, vh, dk, dv, rule, order, counts,
                  fresh=tokens in (2, 33, 64), skip=rule == SELECTIVE or tokens == 5,
                  gate_bias=tokens != 16)
    if ragged:  # rows behind a sequence's are not read
        for s in range(3):
            for x in (scan.q, scan.k, scan.v, scan.gate) + ((scan.beta,) if rule == DELTA else ()):
                x[s, counts[s]:] = np.nan
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan, in_place=tokens % 4 != 0)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
def test_long(hip_ctx, dev, rule):
    """A prompt of many chunks, and heads that share keys in both orders."""
    for order in (0, 1):
        rng = np.random.default_rng(order)
        scan = M.Scan(rng, 2, 1031, 2, 6, 128, 128 if order else 48, rule, order, [1031, 700])
        scan.gate -= 3.0  # states that last
        out, out_tol, state, state_tol = scan.run(chunked=True)
        got, new = run(hip_ctx, dev, scan)
        check_out(got, out, out_tol)
        within(new, state, state_tol, "state")


@pytest.mark.parametrize("tokens", [4, 50])
@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
def test_parts(hip_ctx, dev, rule, tokens):
    """Outputs alone leave the state; the state alone, `more` tokens further than counted."""
    rng = np.random.default_rng(11)
    scan = M.Scan(rng, 3, tokens, 2, 4, 64, 96, rule)
    out, out_tol, state, state_tol = scan.run()
    scan.put(dev)
    o, st = outputs(dev, scan)
    d_out = dev.put(o)
    scan.call(hip_ctx, scan.d_state, None, d_out)
    hip_ctx.synchronize()
    check_out(dev.get(d_out, o), out, out_tol)
    assert np.array_equal(dev.get(scan.d_state, st), scan.state)
    accepted = np.array([0, 2, 0xFFFFFFFF], np.uint32)
    scan.counts = [1, 3, tokens]
    _, _, state, state_tol = scan.run()
    scan.call(hip_ctx, scan.d_state, scan.d_state, None, d_counts=dev.put(accepted), more=1, d_q=None)
    hip_ctx.synchronize()
    within(dev.get(scan.d_state, st), state, state_tol, "state")


def test_nothing_to_do(hip_ctx, dev):
    """Sequences of no tokens: states are copied, outputs stay."""
    rng = np.random.default_rng(12)
    for tokens in (1, 40):
        scan = M.Scan(rng, 2, tokens, 1, 2, 64, 64, counts=[0, 0])
        got, new = run(hip_ctx, dev, scan, in_place=False)
        assert np.all(got == 9.0) and np.array_equal(new, scan.state)
        fresh = M.Scan(rng, 2, tokens, 1, 2, 64, 64, counts=[0, 0], fresh=True)
        got, new = run(hip_ctx, dev, fresh, in_place=False)
        assert np.all(got == 9.0) and np.all(new == 0.0)


@pytest.mark.parametrize("tokens", [3, 80])
def test_in_parts_and_whole(hip_ctx, dev, tokens):
    """Calls of any length from the state of the one before: within both sides' tolerance."""
    rng = np.random.default_rng(13)
    scan = M.Scan(rng, 1, tokens, 2, 4, 128, 64, fresh=True)
    out, out_tol, state, state_tol = scan.run(chunked=True)
    scan.put(dev)
    o, st = outputs(dev, scan)
    d_out, d_state = dev.put(o), dev.put(st)
    t = 0
    while t < tokens:
        n = min((1, 40, 2, 20, 17)[t % 5], tokens - t)
        row = lambda name, size: scan.d[name] + 4 * t * size  # noqa: E731
        hip_ctx.state_scan_device(
            scan.handle, 1, n, row("d_q", scan.stride), row("d_k", scan.stride), row("d_v", scan.stride),
            row("d_gate", 4), row("d_beta", 4), d_state=d_state if t else None, d_state_out=d_state,
            d_out=d_out + 4 * t * 4 * 64, q_token_stride=scan.stride, k_token_stride=scan.stride,
            v_token_stride=scan.stride)
        t += n
    hip_ctx.synchronize()
    check_out(dev.get(d_out, o), out, out_tol)
    within(dev.get(d_state, st), state, state_tol, "state")


@pytest.mark.parametrize("tokens", [12, 70])
@pytest.mark.parametrize("what", ["loud", "shut", "open", "small", "still", "repeat"])
def test_extremes(hip_ctx, dev, what, tokens):
    """Tokens of very different size, gates that clear the state or keep it, equal keys."""
    rng = np.random.default_rng(14)
    scan = M.Scan(rng, 2, tokens, 2, 4, 128, 80)
    if what == "loud":  # one token far above the others, then a gate that forgets it
        scan.v[:, 3] *= 1e12
        scan.gate[:, 4] = 60.0
    elif what == "shut":
        scan.gate[:] = 40.0
        scan.gate[:, ::3] = -40.0
    elif what == "open":
        scan.gate[:] = -60.0
        scan.beta[:] = 30.0
    elif what == "small":
        scan.v *= 1e-30
        scan.state *= np.float32(1e-30)
    elif what == "still":
        scan.beta[:] = -80.0
    else:
        scan.k[:] = scan.k[:, :1]
        scan.beta[:] = 8.0
        scan.gate[:] = -20.0
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("tokens", [9, 75])
@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("what", ["v", "k", "q", "gate", "beta", "state", "v inf", "gate inf"])
def test_numbers_that_are_none(hip_ctx, dev, what, rule, tokens):
    """They reach their own and later tokens' outputs and states, of their column (a value's or a state's)
    or head, and nothing before or beside them."""
    if what == "beta" and rule == SELECTIVE:
        pytest.skip("no such input")
    rng = np.random.default_rng(15)
    scan = M.Scan(rng, 2, tokens, 2, 2, 64, 48, rule)
    clean = scan.run()
    bad_out, bad_state = np.zeros(clean[0].shape, bool), np.zeros(clean[2].shape, bool)
    at = tokens - 4
    if what in ("v", "v inf"):
        scan.v[1, at, 0, 5] = np.nan if what == "v" else np.inf
        bad_out[1, at:, 0, 5] = bad_state[1, 0, :, 5] = True
    elif what == "state":
        scan.state[1, 1, 7, 9] = np.nan
        bad_out[1, :, 1, 9] = bad_state[1, 1, :, 9] = True
    elif what == "q":
        scan.q[1, at, 1, 3] = np.nan
        bad_out[1, at, 1] = True
    else:
        name, _, value = what.partition(" ")
        getattr(scan, name)[(1, at, 0) + ((3,) if name == "k" else ())] = np.inf if value else np.nan
        bad_out[1, at:, 0] = bad_state[1, 0] = True
    got, new = run(hip_ctx, dev, scan)
    within(got[~bad_out], clean[0][~bad_out], clean[1][~bad_out], "out")
    within(new[~bad_state], clean[2][~bad_state], clean[3][~bad_state], "state")
    if what in ("v", "q", "gate", "beta"):
        assert np.all(np.isnan(got[bad_out]))


def test_captured(hip_ctx, dev):
    """A convolution and a scan of a token, in place, captured once and replayed, and the same call by
    call."""
    rng = np.random.default_rng(16)
    kh, vh, dk, dv, width, n = 2, 4, 64, 64, 4, 2
    channels = 2 * kh * dk + vh * dv
    scan = M.Scan(rng, n, 1, kh, vh, dk, dv).put(dev)
    w = rng.standard_normal((channels, width)).astype(np.float32)
    d_w, steps = dev.put(w), 6
    x = rng.standard_normal((steps, n, channels)).astype(np.float32)
    results = []
    for graph in (False, True):
        d_x, d_y = dev.put(x[0]), dev.put(np.zeros((n, channels), np.float32))
        d_conv = dev.put(np.zeros((n, width - 1, channels), np.float32))
        d_state, d_out = dev.put(scan.state), dev.put(np.zeros((n, vh, dv), np.float32))

        def submit():
            hip_ctx.causal_conv_device(d_x, d_w, n, 1, channels, width, d_y=d_y, d_state=d_conv,
                                       d_state_out=d_conv)
            hip_ctx.state_scan_device(
                scan.handle, n, 1, d_y, d_y + 4 * kh * dk, d_y + 8 * kh * dk, scan.d["d_gate"],
                scan.d["d_beta"], d_state=d_state, d_state_out=d_state, d_out=d_out,
                q_token_stride=channels, k_token_stride=channels, v_token_stride=channels)

        if graph:
            hip_ctx.capture_begin()
            submit()
            g = hip_ctx.capture_end()
        made = []
        for t in range(steps):
            hip_ctx.to_device(d_x, x[t])
            g.launch() if graph else submit()
            hip_ctx.synchronize()
            made.append((dev.get(d_out, np.empty((n, vh, dv), np.float32)),
                         dev.get(d_state, scan.state), dev.get(d_conv, np.empty((n, 3, channels), np.float32))))
        results.append(made)
        if graph:
            g.free()
    for a, b in zip(*results):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
    assert not np.array_equal(results[0][0][1], results[0][-1][1])


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
def test_generic_policy(hip_ctx, dev, rule):
    """Prompts token by token, where the tuned kernels are switched off."""
    scan = M.Scan(np.random.default_rng(17), 2, 45, 2, 4, 96, 40, rule, counts=[45, 30])
    out, out_tol, state, state_tol = scan.run(chunked=False)
    hip_ctx.set_kernel_policy(si_hip.KERNEL_GENERIC)
    try:
        got, new = run(hip_ctx, dev, scan)
    finally:
        hip_ctx.set_kernel_policy(si_hip.KERNEL_AUTO)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("heads,sequences,dv", [(4, 2, 128), (64, 3, 128), (70, 6, 128), (70, 6, 40)])
def test_workgroups_of_all_widths(hip_ctx, dev, heads, sequences, dv):
    """Few heads, and as many as take workgroups of four and eight times sixteen columns."""
    scan = M.Scan(np.random.default_rng(heads), sequences, 70, 2, heads, 128, dv,
                  counts=[70, 69, 33, 32, 31, 1][:sequences])
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


def test_rows_far_apart(hip_ctx, dev):
    """Rows a stride that no chunk's buffer reaches over are taken token by token."""
    rng = np.random.default_rng(18)
    scan = M.Scan(rng, 1, 9, 1, 1, 32, 16)
    out, out_tol, state, state_tol = scan.run(chunked=False)
    scan.put(dev)
    stride = (1 << 23) + 4
    far = dev.raw(4 * (8 * stride + 32))
    for t in range(9):
        hip_ctx.to_device(far + 4 * t * stride, scan.k[0, t])
    o, st = outputs(dev, scan)
    d_out = dev.put(o)
    scan.call(hip_ctx, scan.d_state, scan.d_state, d_out, d_k=far, k_token_stride=stride)
    hip_ctx.synchronize()
    check_out(dev.get(d_out, o), out, out_tol)
    within(dev.get(scan.d_state, st), state, state_tol, "state")


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("tokens", [3, 50])
def test_states_that_fade_and_grow(hip_ctx, dev, tokens, rule):
    """Columns from 1e-36 to 1e30 beside one another, states that all but vanish, and units that follow.

    A chunk's factors e^(G_i - G_j) are f32 numbers, those below 2^-126 count as zero. With M no less than
    the norms of a column's states and its |u|, keys and queries of length 1 and w < 1, each R_i is off by at
    most 2^-126 M for its state and 31 * 2^-126 M for its row of L: by 2^-121 M. The system takes these as it
    takes values, and I - w k k^T lengthens nothing: 32 of them put at most 2^-116 M into the states
    and outputs of a chunk, P's own factors and the state's 33 * 2^-126 M. Entries of the inverse
    and the sums of up to 32 products that make them lose 2^-126 as often: 2^-115 M a chunk, and 2^-114 M
    for two chunks.  (The selective form has neither the system nor such lengths: there M takes those of keys
    and queries.)"""
    rng = np.random.default_rng(19)
    scan = M.Scan(rng, 2, tokens, 1, 2, 64, 64, rule)
    size = np.float32(10.0) ** np.linspace(-36, 30, 64).astype(np.float32)
    scan.v *= size
    scan.state *= size[::-1]
    scan.gate[0] += 6.0
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    largest = (np.sqrt((scan.state.astype(np.float64) ** 2).sum(2)).max(1)
               + np.abs(scan.v.astype(np.float64)).sum(1).max(1))
    if rule == SELECTIVE:
        length = lambda x: np.maximum(1, np.sqrt((x.astype(np.float64) ** 2).sum(-1)).max())  # noqa: E731
        largest *= length(scan.k) * length(scan.q * scan.scale) * 8  # (and steps of up to 8)
    # (below 1e-30 a value has fewer bits, down to the least numbers of f32)
    lost = 1e-37 + (2.0 ** -114 * largest if tokens >= 4 else 0 * largest)
    check_out(got, out, out_tol + lost[:, None, None])
    within(new, state, state_tol + lost[:, None, None], "state")


def test_outputs_apart_from_inputs(hip_ctx):
    """Refused before anything runs: outputs that are one of the inputs (none of the pointers is read)."""
    p, lib = [4096 * (i + 1) for i in range(9)], si_hip.lib()
    q, k, v, gate, beta, state, decay = p[:7]
    scan = si_hip.StateScan(rule=0, head_order=0, key_heads=1, value_heads=1, key_dim=32, value_dim=32,
                            scale=1.0, eps=1e-6, d_decay=decay)

    def call(state_out, out):
        return lib.si_hip_state_scan_device(hip_ctx.handle, scan, 1, 1, None, 0, q, 32, k, 32, v, 32, gate, beta,
                                            state, state_out, out)

    for x in (q, k, v, gate, beta):
        assert call(x, p[8]) != 0 and "writes what it reads" in si_hip.last_error()
        assert call(p[8], x) != 0 and "writes what it reads" in si_hip.last_error()
    assert call(state, state) != 0 and call(p[8], p[8]) != 0
    assert "writes what it reads" in si_hip.last_error()

    def conv(x, state, state_out, y):
        return lib.si_hip_causal_conv_device(hip_ctx.handle, 1, 1, None, 0, 32, 4, x, 32, decay, None, 0, state,
                                             state_out, y, 32)

    for args in ((q, state, state, q), (q, state, q, k), (q, k, state, k), (q, state, k, k)):
        assert conv(*args) != 0 and "writes what it reads" in si_hip.last_error()


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("dk", [132, 160, 161, 192, 200, 256])
@pytest.mark.parametrize("heads,sequences,dv,tokens", [(2, 2, 64, 100), (64, 3, 72, 40), (1, 1, 256, 300)])
def test_many_keys(hip_ctx, dev, dk, heads, sequences, dv, tokens, rule):
    """Heads of more than 128 keys, whose chunks have fewer buffers, by workgroups of both widths."""
    scan = M.Scan(np.random.default_rng(dk + tokens), sequences, tokens, 1, heads, dk, dv, rule,
                  counts=[tokens, tokens // 3, 32][:sequences])
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("where", ["q", "k", "v", "gate", "beta"])
def test_numbers_that_are_none_many_keys(hip_ctx, dev, where):
    """Tokens before one that is none, other heads and other sequences are what they are without it."""
    scan = M.Scan(np.random.default_rng(23), 2, 70, 2, 2, 256, 40)
    out, out_tol, state, state_tol = scan.run()
    getattr(scan, where)[1, 37, 1] = np.nan
    got, new = run(hip_ctx, dev, scan)
    bad_out, bad_state = np.zeros(out.shape, bool), np.zeros(state.shape, bool)
    bad_out[1, 37:38 if where == "q" else None, 1] = True
    bad_state[1, 1] = where != "q"
    within(got[~bad_out], out[~bad_out], out_tol[~bad_out], "out")
    within(new[~bad_state], state[~bad_state], state_tol[~bad_state], "state")
    assert np.all(np.isnan(got[bad_out]))


@pytest.mark.parametrize("what", ["v", "k"])
@pytest.mark.parametrize("heads,sequences", [(64, 3), (70, 6)])
def test_numbers_that_are_none_many_heads(hip_ctx, dev, heads, sequences, what):
    """The same in workgroups of four and eight times sixteen columns."""
    scan = M.Scan(np.random.default_rng(29), sequences, 50, 2, heads, 128, 128)
    out, out_tol, state, state_tol = scan.run()
    bad_out, bad_state = np.zeros(out.shape, bool), np.zeros(state.shape, bool)
    if what == "v":
        scan.v[1, 40, 5, 77] = np.nan
        bad_out[1, 40:, 5, 77] = bad_state[1, 5, :, 77] = True
    else:
        scan.k[1, 40, 1, 100] = np.inf  # of the second half of the heads
        bad_out[1, 40:, heads // 2:] = bad_state[1, heads // 2:] = True
    got, new = run(hip_ctx, dev, scan)
    within(got[~bad_out], out[~bad_out], out_tol[~bad_out], "out")
    within(new[~bad_state], state[~bad_state], state_tol[~bad_state], "state")
    if what == "v":
        assert np.all(np.isnan(got[bad_out])) and np.all(np.isnan(new[bad_state]))


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("tokens,dk", [(3, 64), (80, 64), (80, 160)])
def test_states_that_grow(hip_ctx, dev, tokens, dk, rule):
    """A decay above zero, and no eps (the tolerances' recurrences hold for any a)."""
    scan = M.Scan(np.random.default_rng(31), 2, tokens, 1, 3, dk, 32, rule)
    scan.decay = np.array([0.5, 0.05, -0.5], np.float32)
    scan.eps = 0.0
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


def test_rows_behind_2_to_32(hip_ctx, dev):
    """Rows as far apart as a chunk's buffers reach, the last ones 2^32 values behind the first."""
    tokens, stride, dim = 515, 1 << 23, 32
    scan = M.Scan(np.random.default_rng(37), 1, tokens, 1, 1, dim, dim)
    scan.gate -= 2.0
    out, out_tol, state, state_tol = scan.run()
    scan.put(dev)
    rows = dev.raw(4 * ((tokens - 1) * stride + 3 * dim))
    for t in range(tokens):
        hip_ctx.to_device(rows + 4 * t * stride,
                          np.concatenate([scan.q[0, t, 0], scan.k[0, t, 0], scan.v[0, t, 0]]))
    o, st = outputs(dev, scan)
    d_out = dev.put(o)
    scan.call(hip_ctx, scan.d_state, scan.d_state, d_out, d_q=rows, d_k=rows + 4 * dim, d_v=rows + 8 * dim,
              q_token_stride=stride, k_token_stride=stride, v_token_stride=stride)
    hip_ctx.synchronize()
    check_out(dev.get(d_out, o), out, out_tol)
    within(dev.get(scan.d_state, st), state, state_tol, "state")


@pytest.mark.parametrize("gate", [1e9, 1e12, 1e14, 1e16, 1e30, 3e38, np.inf])
@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("tokens,at,dk", [(3, 1, 64), (12, 3, 64), (70, 40, 128), (70, 37, 160)])
def test_gates_that_clear_the_state(hip_ctx, dev, tokens, at, dk, rule, gate):
    """A gate so large that nothing before its token is left, in the middle of a chunk, and ordinary ones
    behind it: what follows is a sequence that begins there, without a state.  (So the reference's first
    token needs no such gate; the selective form's step multiplies the value, too, which is made that
    much smaller, and so rounded once more, and has no product with an infinite one.)"""
    if rule == SELECTIVE and gate == np.inf:
        pytest.skip("its step times a value is no finite number")
    scan = M.Scan(np.random.default_rng(41), 2, tokens, 1, 3, dk, 48, rule)
    whole = scan.run()
    rest = copy.copy(scan)
    rest.shape = (2, tokens - at) + scan.shape[2:]
    for name in ("q", "k", "v", "gate", "beta"):
        x = getattr(scan, name)
        setattr(rest, name, None if x is None else x[:, at:].copy())
    rest.state = None
    rest.gate[:, 0] = 0.0
    scan.gate[:, at] = gate
    if rule == SELECTIVE:
        scan.v[:, at] /= np.float32(gate)
        step = np.logaddexp(0.0, rest.bias.astype(np.float64))
        rest.v[:, 0] = (scan.v[:, at].astype(np.float64) * np.float64(np.float32(gate)) / step[:, None])
    out, out_tol, state, state_tol = rest.run(chunked=tokens >= 4)
    got, new = run(hip_ctx, dev, scan)
    within(got[:, :at], whole[0][:, :at], whole[1][:, :at], "out before")
    within(got[:, at:], out, out_tol, "out behind")
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("eps", [1e-6, 1.0])
@pytest.mark.parametrize("size", [1e-4, 1e-7, 1e-9, 1e-12, 1e-20, 1e-30])
@pytest.mark.parametrize("tokens,dk,which", [(6, 64, "q"), (40, 128, "q"), (40, 160, "q"), (6, 64, "k"),
                                             (40, 128, "k"), (70, 33, "k"), (40, 160, "k"), (70, 64, "qk")])
def test_short_rows(hip_ctx, dev, tokens, dk, which, size, eps):
    """Keys and queries far shorter than eps's root, some of them or all of a chunk's, zeros among them: their
    products are as exact as longer ones', to the least numbers of f32 and their products."""
    rng = np.random.default_rng(43)
    scan = M.Scan(rng, 2, tokens, 2, 4, dk, 40)
    scan.eps = eps
    scan.gate -= 2.0
    rows = np.ones(tokens, bool)
    if tokens != 40:
        rows[1::3] = False
    for name in which:
        x = getattr(scan, name)
        x[:, rows] *= np.float32(size)
        x[:, 3] = 0.0
    if "k" in which:  # so that what such keys leave is what the outputs are made of
        scan.state[:] = 0.0
        scan.v *= np.float32(min(1.0 / size, 1e12))
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("tokens", [1, 40])
def test_outputs_behind_the_inputs(hip_ctx, dev, tokens):
    """A buffer that ends where the next begins; without outputs, queries that are the state."""
    scan = M.Scan(np.random.default_rng(47), 1, tokens, 2, 4, 64, 32)
    out, out_tol, state, state_tol = scan.run()
    scan.put(dev)
    rows = np.concatenate([x.reshape(tokens, -1) for x in (scan.q, scan.k, scan.v)], 1)
    space = np.zeros(rows.size + out.size + scan.state.size, np.float32)
    space[:rows.size], space[rows.size + out.size:] = rows.reshape(-1), scan.state.reshape(-1)
    d = dev.put(space)
    at = dict(d_q=d, d_k=d + 4 * 128, d_v=d + 8 * 128)
    d_out, d_state = d + 4 * rows.size, d + 4 * (rows.size + out.size)
    scan.call(hip_ctx, d_state, None, d_out, **at)
    scan.call(hip_ctx, d_state, d_state, None, **{**at, "d_q": d_state})
    hip_ctx.synchronize()
    got = dev.get(d, space)
    assert np.array_equal(got[:rows.size], space[:rows.size])
    check_out(got[rows.size:rows.size + out.size].reshape(out.shape), out, out_tol)
    within(got[rows.size + out.size:].reshape(state.shape), state, state_tol, "state")


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("dk,dv", [(32, 64), (64, 64), (64, 72), (64, 128), (128, 120), (128, 128)])
def test_short_calls_of_many_heads(hip_ctx, dev, dk, dv, rule):
    """Around the lengths from which calls of several rounds are taken in chunks."""
    for tokens in (7, 8, 11, 12, 15, 16):
        scan = M.Scan(np.random.default_rng(tokens), 6, tokens, 2, 90, dk, dv, rule,
                      counts=[tokens, 0, tokens - 1, 1, tokens, tokens])
        out, out_tol, state, state_tol = scan.run()
        got, new = run(hip_ctx, dev, scan)
        check_out(got, out, out_tol)
        within(new, state, state_tol, "state")


@pytest.mark.parametrize("loud", [1.0, 1e5, 1e12, 1e25])
@pytest.mark.parametrize("tokens,dk,heads,sequences", [(3, 64, 4, 2), (12, 64, 4, 2), (70, 128, 4, 2), (70, 160, 4, 2),
                                                       (40, 128, 70, 6)])
def test_zero_keys(hip_ctx, dev, tokens, dk, heads, sequences, loud):
    """Tokens whose keys are zeros leave the state what it is, whatever their values are."""
    scan = M.Scan(np.random.default_rng(53), sequences, tokens, 2, heads, dk, 72)
    scan.gate -= 3.0
    scan.k[:, 1::3, 0] = 0.0
    scan.v[:, 1::3, :heads // 2] *= np.float32(loud)  # of the heads that share these keys
    scan.k[0, :, 1] = 0.0
    scan.v[0, :, heads // 2:] *= np.float32(loud)
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")


@pytest.mark.parametrize("rule", [DELTA, SELECTIVE])
@pytest.mark.parametrize("tokens,dk,heads,sequences", [(3, 64, 4, 2), (70, 33, 6, 2), (70, 128, 6, 2), (40, 160, 4, 2),
                                                       (40, 128, 70, 6)])
def test_outputs_that_are_their_inputs(hip_ctx, dev, tokens, dk, heads, sequences, rule):
    """Outputs of which skip v is all but a little: to the two roundings of f32 that put it there."""
    scan = M.Scan(np.random.default_rng(59), sequences, tokens, 2, heads, dk, 72, rule, skip=True)
    scan.scale = float(np.float32(1e-6))
    out, out_tol, state, state_tol = scan.run()
    got, new = run(hip_ctx, dev, scan)
    check_out(got, out, out_tol)
    within(new, state, state_tol, "state")
