"""CPU: refusals of a hybrid decoder layer's mixers (include/si_hip_mixer.h, the head norms and
several-axis positions of include/si_hip_decode.h), each before the context is looked at, and the
table of axes."""
import ctypes as C

import numpy as np
import pytest

import si_hip
from test_decode_abi import DIM, NULL, OVER, P, RANGE, TYPE, BATCH, cache, rope

NAN, INF = float("nan"), float("inf")


def norm(**more):
    return si_hip.HeadNorm(**{**dict(eps=1e-6, plus_one=0, d_q_weight=P, d_k_weight=P), **more})


def axes(**more):
    return si_hip.RopeAxes(**{**dict(axes=3, d_axis=P), **more})


def rows(n="norm", r="rope", a=None, x=P, tokens=3, heads=8, dim=64, ts=512, hs=64, pos=P, y=P + 64,
         yts=512, yhs=64):
    return si_hip.lib().si_hip_norm_rope_device(
        None, norm() if n == "norm" else n, rope() if r == "rope" else r, a, x, tokens, heads, dim, ts,
        hs, pos, y, yts, yhs)


def append(c=None, n="norm", r="rope", a=None, tokens=1, k=P, ks=256, v=P, vs=256, q=None, heads=8,
           qs=512, qh=64, qo=P + 64):
    return si_hip.lib().si_hip_norm_rope_append_device(
        None, c or cache(), norm() if n == "norm" else n, rope() if r == "rope" else r, a, tokens, None,
        None, k, ks, v, vs, q, heads, qs, qh, qo)


@pytest.mark.parametrize("call", [rows, append])
def test_norm_and_axes(call):
    assert call() == NULL and "argument is null" in si_hip.last_error()  # only the context is missing
    for more in (dict(eps=0.0), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF), dict(plus_one=2)):
        assert call(n=norm(**more)) == DIM
        assert "head norm" in si_hip.last_error()
    assert call(n=norm(d_q_weight=None, d_k_weight=None)) == NULL
    assert "argument is null" in si_hip.last_error()
    for more in (dict(axes=0), dict(axes=5)):
        assert call(a=axes(**more)) == DIM
    assert call(a=axes(d_axis=None)) == NULL and "axis table" in si_hip.last_error()
    assert call(a=axes(), r=None) == NULL and "axes need" in si_hip.last_error()
    assert call(r=rope(layout=2)) == TYPE and call(r=rope(rotary_dim=66)) == DIM
    assert call(r=rope(d_frequencies=None)) == NULL


def test_rows():
    assert rows(n=None, r=None) == NULL and "neither" in si_hip.last_error()
    assert rows(n=None) == NULL and rows(r=None, pos=None) == NULL
    assert rows(tokens=0) == DIM and rows(heads=0) == DIM and rows(dim=0) == DIM and rows(dim=257) == DIM
    assert rows(tokens=1 << 31) == OVER and rows(heads=1 << 16, ts=1 << 40, yts=1 << 40) == OVER
    assert rows(ts=511) == DIM and rows(hs=63) == DIM and rows(yts=511) == DIM and rows(yhs=63) == DIM
    assert rows(hs=1 << 62, ts=1 << 62) == OVER


def test_append():
    assert append(tokens=0) == BATCH
    assert append(cache(ggml_type=2)) == TYPE and append(cache(head_dim=300)) == DIM
    assert append(cache(sequences=60000), tokens=1 << 20) == OVER
    assert append(ks=255) == DIM and append(vs=255) == DIM
    assert append(q=P, heads=6) == DIM and append(q=P, qs=511) == DIM and append(q=P, qh=63) == DIM
    assert append(q=P, qo=None) == NULL
    assert append(q=P, n=None, r=None) == NULL and "query rows need" in si_hip.last_error()
    assert append(q=P, qo=P, qs=1024, qh=128) == DIM and "contiguous" in si_hip.last_error()
    assert append(k=None) == NULL and append(v=None) == NULL and append(n=None, r=None) == NULL


def table(rotary, sections, order):
    return si_hip.rope_axis_table(rotary, sections, order)


def test_axis_table():
    assert list(table(16, [8], 0)) == [0] * 8 and list(table(16, [8], 1)) == [0] * 8
    assert list(table(16, [3, 0, 5], 0)) == [0] * 3 + [2] * 5
    assert list(table(16, [0, 3, 5], 0)) == [1] * 3 + [2] * 5
    got = list(table(128, [24, 20, 20], 1))
    assert got[:60] == [0, 1, 2] * 20 and got[60:] == [0] * 4
    assert list(table(64, [11, 11, 10], 1)) == [0, 1, 2] * 10 + [0, 1]
    assert list(table(8, [1, 1, 1, 1], 1)) == [0, 1, 2, 3]
    for rotary, sections, order, status in [
            (16, [8], 2, TYPE), (0, [0], 0, DIM), (15, [7], 0, DIM), (258, [129], 0, DIM),
            (16, [], 0, DIM), (16, [2] * 5, 0, DIM), (16, [7], 0, DIM), (16, [4, 5], 0, DIM),
            (16, [1, 7], 1, DIM), (16, [0, 4, 4], 1, DIM), (16, [1 << 31, (1 << 31) + 8], 0, DIM)]:
        with pytest.raises(si_hip.HipError) as e:
            table(rotary, sections, order)
        assert e.value.status == status, (rotary, sections, order)
    assert si_hip.lib().si_hip_rope_axis_table(16, None, 1, 0, None) == NULL


def conv(sequences=2, tokens=3, counts=None, more=0, channels=40, width=4, x=P, xs=40, w=P, b=None,
         act=1, state=P, out=P, y=P + 64, ys=40):
    return si_hip.lib().si_hip_causal_conv_device(
        None, sequences, tokens, counts, more, channels, width, x, xs, w, b, act, state, out, y, ys)


def test_conv():
    assert conv() == NULL
    assert conv(sequences=0) == DIM and conv(tokens=0) == DIM and conv(more=1) == DIM
    assert conv(counts=P, more=1) == NULL
    assert conv(sequences=65536) == OVER and conv(sequences=60000, tokens=1 << 20) == OVER
    assert conv(act=2) == TYPE
    assert conv(channels=0) == DIM and conv(width=1) == DIM and conv(width=9) == DIM and conv(width=8) == NULL
    assert conv(channels=1 << 31, xs=1 << 31, ys=1 << 31) == OVER
    assert conv(xs=39) == DIM and conv(ys=39) == DIM and conv(y=None, ys=0) == NULL
    assert conv(xs=1 << 40) == OVER
    assert conv(x=None) == NULL and conv(w=None) == NULL and conv(y=None, out=None) == NULL


def scan(h=None, sequences=2, tokens=3, counts=None, more=0, q=P, qs=128, k=P, ks=128, v=P, vs=192,
         gate=P, beta=P, state=P, state_out=P, out=P + 64):
    return si_hip.lib().si_hip_state_scan_device(
        None, h or shape(), sequences, tokens, counts, more, q, qs, k, ks, v, vs, gate, beta, state,
        state_out, out)


def shape(**more):
    return si_hip.StateScan(**{**dict(rule=0, head_order=0, key_heads=2, value_heads=4, key_dim=64,
                                      value_dim=48, scale=0.125, eps=1e-6, d_decay=P), **more})


def test_scan():
    assert scan() == NULL and "argument is null" in si_hip.last_error()
    assert si_hip.lib().si_hip_state_scan_device(None, None, *[0] * 15) == NULL
    assert scan(shape(rule=2)) == TYPE and scan(shape(head_order=2)) == TYPE
    for more in (dict(key_heads=0), dict(value_heads=0), dict(key_heads=3), dict(key_dim=0),
                 dict(key_dim=257), dict(value_dim=0), dict(value_dim=257), dict(scale=NAN),
                 dict(scale=INF), dict(eps=-1e-9), dict(eps=NAN)):
        assert scan(shape(**more)) == DIM, more
    assert scan(shape(rule=1, eps=NAN), beta=None) == NULL
    assert scan(shape(key_heads=1, value_heads=65536), vs=1 << 23) == OVER
    assert scan(sequences=0) == DIM and scan(tokens=0) == DIM and scan(more=2) == DIM
    assert scan(sequences=70000) == OVER and scan(sequences=60000, tokens=60000) == OVER
    assert scan(qs=127) == DIM and scan(ks=127) == DIM and scan(vs=191) == DIM
    assert scan(qs=0, q=None, out=None) == NULL
    for more in (dict(k=None), dict(v=None), dict(gate=None), dict(beta=None), dict(q=None),
                 dict(out=None, state_out=None)):
        assert scan(**more) == NULL
    # (with a context those are refused, too: the outputs are none of the inputs)


# Refusals of outputs that share memory with what a call reads come last, so they need a context: this one is
# never looked at.
FAKE = C.create_string_buffer(1 << 16)
CONTEXT = C.addressof(FAKE)
ROOM = 1 << 20  # bytes between arguments that share nothing


def shared(status):
    return status == RANGE and "writes what it reads" in si_hip.last_error()


CONV = dict(sequences=3, tokens=5, counts=2, channels=40, width=4, xs=90, ys=100)


def conv_at(**more):
    a = {**{k: ROOM * (i + 1) for i, k in enumerate(("x", "w", "b", "state", "out", "y", "n"))}, **CONV, **more}
    return si_hip.lib().si_hip_causal_conv_device(
        CONTEXT, a["sequences"], a["tokens"], a["n"], 0, a["channels"], a["width"], a["x"], a["xs"], a["w"], a["b"],
        1, a["state"], a["out"], a["y"], a["ys"])


SIZES = dict(x=4 * (14 * 90 + 40), w=4 * 160, b=160, state=4 * 9 * 40, n=12)


@pytest.mark.parametrize("read", ["x", "w", "b", "state", "n"])
@pytest.mark.parametrize("written,size", [("y", 4 * (14 * 100 + 40)), ("out", 4 * 9 * 40)])
def test_conv_outputs_apart(read, written, size):
    """At the first byte that is shared and the last, from either side."""
    at = 64 * ROOM
    for where in (at, at + 4, at + SIZES[read] - 4, at - size + 4):
        if (read, written, where) != ("state", "out", at):
            assert shared(conv_at(**{read: at, written: where})), where
    assert shared(conv_at(y=at, out=at + 4 * 14 * 100))


def test_conv_in_one_buffer():
    """Rows beside one another in wider ones: a channel that both have, and outputs of another row length."""
    at = 64 * ROOM
    for y in (at + 4 * 39, at + 4 * 91, at + 4 * 90 * 3 - 4, at - 4):
        assert shared(conv_at(x=at, y=y, ys=90))
    assert shared(conv_at(x=at, y=at + 4 * 50, ys=100)) and shared(conv_at(x=at, y=at + 4 * 45, ys=91))
    assert shared(conv_at(x=at, out=at + 4 * 40, channels=40))


SCAN = dict(sequences=3, tokens=5, qs=150, ks=160, vs=210, rule=0)
SCAN_SIZES = dict(q=4 * (14 * 150 + 128), k=4 * (14 * 160 + 128), v=4 * (14 * 210 + 192), gate=4 * 60, beta=4 * 60,
                  state=4 * 3 * 4 * 64 * 48, decay=16, bias=16, skip=16, n=12, state_out=4 * 3 * 4 * 64 * 48,
                  out=4 * 15 * 192)


def scan_at(**more):
    a = {**{k: ROOM * (i + 1) for i, k in enumerate(SCAN_SIZES)}, **SCAN, **more}
    h = shape(d_decay=a["decay"], d_bias=a["bias"], d_skip=a["skip"], rule=a["rule"])
    return si_hip.lib().si_hip_state_scan_device(
        CONTEXT, h, a["sequences"], a["tokens"], a["n"], 0, a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["gate"],
        a["beta"], a["state"], a["state_out"], a["out"])


@pytest.mark.parametrize("read", ["q", "k", "v", "gate", "beta", "decay", "bias", "skip", "n", "state"])
@pytest.mark.parametrize("written", ["out", "state_out"])
def test_scan_outputs_apart(read, written):
    """At the first byte that is shared and the last, from either side."""
    at = 64 * ROOM
    for where in (at, at + 4, at + SCAN_SIZES[read] - 4, at - SCAN_SIZES[written] + 4):
        if (read, written, where) != ("state", "state_out", at):
            assert shared(scan_at(**{read: at, written: where})), where
    assert shared(scan_at(out=at, state_out=at + SCAN_SIZES["out"] - 4))


def test_scan_in_one_buffer():
    """Queries, keys and values in the rows of one buffer, and an output that begins among them."""
    at = 64 * ROOM
    qkv = dict(q=at, k=at + 4 * 128, v=at + 8 * 128, qs=448, ks=448, vs=448)
    for more in (dict(out=at + 8 * 128 + 4), dict(out=at + 4 * 448), dict(state_out=at + 4 * 447)):
        assert shared(scan_at(**qkv, **more))
    assert shared(scan_at(rule=1, beta=None, gate=at, out=at + 236))


ROWS_SIZES = dict(x=4 * (2 * 700 + 7 * 80 + 64), qw=256, freq=256, axis=32, pos=4 * 9)


def rows_at(**more):
    a = {**{k: ROOM * (i + 1) for i, k in enumerate([*ROWS_SIZES, "kw", "y"])},
         **dict(ts=700, hs=80, yts=900, yhs=96, one=False), **more}
    return si_hip.lib().si_hip_norm_rope_device(
        CONTEXT, norm(d_q_weight=a["qw"], d_k_weight=a["kw"]), rope(d_frequencies=a["freq"]),
        None if a["one"] else axes(d_axis=a["axis"]), a["x"], 3, 8, 64, a["ts"], a["hs"], a["pos"], a["y"], a["yts"],
        a["yhs"])


@pytest.mark.parametrize("read", ROWS_SIZES)
def test_rows_outputs_apart(read):
    at, size = 64 * ROOM, 4 * (2 * 900 + 7 * 96 + 64)
    for where in (at, at + 4, at + ROWS_SIZES[read] - 4, at - size + 4):
        if (read, where) != ("x", at):
            assert shared(rows_at(**{read: at, "y": where})), where
    assert shared(rows_at(x=at, y=at + 4, yts=700, yhs=80)) and shared(rows_at(x=at, y=at + 4 * 79, yts=700, yhs=80))
    assert shared(rows_at(pos=at, y=at - size + 4, one=True)) and rows_at(x=at, y=at) == DIM


APPEND_SIZES = dict(k=4 * (5 * 300 + 256), v=4 * (5 * 310 + 256), q=4 * (5 * 1300 + 7 * 128 + 64), pos=72, qw=256,
                    kw=256, freq=256, axis=32, n=8, table=32, lengths=8)


def append_at(**more):
    a = {**{k: ROOM * (i + 1) for i, k in enumerate([*APPEND_SIZES, "qo"])}, **dict(ks=300, vs=310, qs=1300, qh=128),
         **more}
    return si_hip.lib().si_hip_norm_rope_append_device(
        CONTEXT, cache(d_page_table=a["table"], d_lengths=a["lengths"]), norm(d_q_weight=a["qw"], d_k_weight=a["kw"]),
        rope(d_frequencies=a["freq"]), axes(d_axis=a["axis"]), 3, a["n"], a["pos"], a["k"], a["ks"], a["v"], a["vs"],
        a["q"], 8, a["qs"], a["qh"], a["qo"])


@pytest.mark.parametrize("read", APPEND_SIZES)
def test_append_outputs_apart(read):
    at, size = 64 * ROOM, 4 * 6 * 512
    for where in (at, at + 4, at + APPEND_SIZES[read] - 4, at - size + 4):
        if (read, where) != ("q", at):
            assert shared(append_at(**{read: at, "qo": where})), where
    assert append_at(q=at, qo=at) == DIM
    # q, k and v in one row, the outputs among them
    row = dict(q=at, qs=1100, qh=64, k=at + 2064, ks=1100, v=at + 3100, vs=1100)
    assert shared(append_at(**row, qo=at + 4400 * 5 + 2064)) and shared(append_at(**row, qo=at + 4400 * 5 + 4120))


@pytest.mark.parametrize("call", [rows, append])
def test_reserved_of_axes(call):
    assert call(a=axes(reserved=1)) == DIM and "rotary axes" in si_hip.last_error()
    assert call(a=axes(axes=1)) == NULL and "argument is null" in si_hip.last_error()
