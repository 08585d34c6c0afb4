"""CPU: refusals of the decode-step operators (include/si_hip_decode.h), each
before the context is looked at, and the rotary frequency table."""
import ctypes as C

import numpy as np
import pytest

import decode_ref as R
import si_hip

NULL, DIM, LEN, OVER, TYPE, BATCH, RANGE = -1, -2, -3, -4, -5, -6, -7
P = 0x1000  # an address that no call gets to


def cache(**more):
    d = dict(ggml_type=1, kv_heads=4, head_dim=64, page_tokens=16, pages=8, sequences=2, max_pages=4,
             d_keys=P, d_values=P, d_page_table=P, d_lengths=P)
    return si_hip.KvCache(**{**d, **more})


def rope(**more):
    return si_hip.Rope(**{**dict(layout=0, rotary_dim=64, magnitude=1.0, d_frequencies=P), **more})


def append(c=None, r=None, tokens=1, k=P, ks=256, v=P, vs=256, q=None, heads=8, qs=512, qh=64, qo=P,
           no_rope=False):
    return si_hip.lib().si_hip_rope_append_device(
        None, c or cache(), None if no_rope else r or rope(), tokens, None, None, k, ks, v, vs, q,
        heads, qs, qh, qo)


def attend(c=None, heads=8, tokens=1, window=0, scale=0.125, q=P, qs=512, qh=64, out=P, w=None, ws=0,
           space=P, size=1 << 30):
    return si_hip.lib().si_hip_paged_attention_device(
        None, c or cache(), heads, tokens, window, scale, None, q, qs, qh, out, w, ws, space, size)


def evict(c=None, w=P, ws=64, keep=16, sinks=2, recent=4, to=None, tw=P + 64, tws=64, kept=P):
    return si_hip.lib().si_hip_kv_evict_device(
        None, c or cache(), w, ws, keep, sinks, recent,
        to or cache(d_page_table=P + 64, d_lengths=P + 64), tw, tws, kept)


@pytest.mark.parametrize("more,status", [
    (dict(ggml_type=2), TYPE), (dict(ggml_type=12), TYPE), (dict(kv_heads=0), DIM),
    (dict(head_dim=0), DIM), (dict(head_dim=257), DIM), (dict(page_tokens=0), DIM),
    (dict(pages=0), DIM), (dict(sequences=0), DIM), (dict(max_pages=0), DIM),
    (dict(max_pages=1 << 28), OVER), (dict(pages=1 << 27), OVER), (dict(kv_heads=70000), OVER),
    (dict(sequences=70000), OVER)])
def test_cache_shapes(more, status):
    c = cache(**more)
    lib = si_hip.lib()
    assert append(c) == status
    assert "key-value cache" in si_hip.last_error()
    assert attend(c) == status and evict(c) == status and evict(to=c) == status
    assert lib.si_hip_kv_advance_device(None, c, None, 1) == status
    assert lib.si_hip_paged_attention_workspace(c, 8, 1, 0) == 0
    assert append() == NULL and attend() == NULL and evict() == NULL  # valid: only the context is missing
    assert lib.si_hip_kv_advance_device(None, cache(), None, 1) == NULL
    assert lib.si_hip_kv_advance_device(None, None, None, 1) == NULL


def test_append_refusals():
    assert append(tokens=0) == BATCH
    assert append(cache(sequences=60000), tokens=1 << 20) == OVER
    assert append(r=rope(layout=2)) == TYPE
    for more in (dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=66),
                 dict(magnitude=float("nan")), dict(magnitude=float("inf"))):
        assert append(r=rope(**more)) == DIM
    assert append(r=rope(d_frequencies=None)) == NULL
    assert append(ks=255) == DIM and append(vs=255) == DIM
    assert append(q=P, heads=6) == DIM and append(q=P, heads=0) == DIM
    assert append(q=P, qs=511) == DIM and append(q=P, qh=63) == DIM
    assert append(q=P, qh=1 << 62) == OVER
    assert append(q=P, qo=None) == NULL and append(q=P, no_rope=True) == NULL
    assert append(q=P, qs=1024, qh=128, qo=P) == DIM
    assert "in place" in si_hip.last_error()
    assert append(k=None) == NULL and append(v=None) == NULL


def test_rope_refusals():
    f = si_hip.lib().si_hip_rope_device
    ok = [None, rope(), P, 3, 8, 64, 512, 64, P, P, 512, 64]
    def call(**at):
        a = list(ok)
        for k, v in at.items():
            a[int(k[1:])] = v
        return f(*a)
    assert call() == NULL
    assert call(a1=None) == NULL
    assert call(a3=0) == DIM and call(a4=0) == DIM and call(a5=0) == DIM and call(a5=300) == DIM
    assert call(a5=32) == DIM  # fewer values than rotate
    assert call(a3=1 << 32) == OVER and call(a4=1 << 17, a6=1 << 40) == OVER
    assert call(a6=511) == DIM and call(a7=63) == DIM and call(a10=511) == DIM and call(a11=63) == DIM
    assert call(a1=rope(layout=3)) == TYPE


def test_attention_refusals():
    assert attend(tokens=0) == BATCH and attend(tokens=17) == BATCH
    assert attend(heads=0) == DIM and attend(heads=6) == DIM
    assert attend(qs=511) == DIM and attend(qh=63) == DIM
    assert attend(scale=float("nan")) == DIM and attend(scale=float("inf")) == DIM
    assert attend(w=P, ws=63) == DIM
    size = si_hip.lib().si_hip_paged_attention_workspace(cache(), 8, 1, 1)
    assert size >= 2 * 8 * 64 * 4
    assert attend(w=P, ws=64, size=size - 1) == LEN
    assert attend(w=P, ws=64, size=size) == NULL
    for t in (0, 17):
        assert si_hip.lib().si_hip_paged_attention_workspace(cache(), 8, t, 0) == 0
    assert si_hip.lib().si_hip_paged_attention_workspace(cache(), 6, 1, 0) == 0


def test_attention_scores_beyond_the_address_space():
    """Sizes whose product wraps to a small workspace."""
    c = cache(sequences=65535, kv_heads=1, max_pages=(1 << 26) + 1, head_dim=1)
    lib = si_hip.lib()
    assert lib.si_hip_paged_attention_workspace(c, 65535, 16, 1) == 0
    assert "attention weights" in si_hip.last_error()
    assert attend(c, heads=65535, tokens=16, qs=65535, qh=1, w=P, ws=1 << 31) == OVER
    assert lib.si_hip_paged_attention_workspace(c, 65535, 16, 0) > 0


def test_evict_refusals():
    assert evict(keep=0) == DIM and evict(keep=65) == DIM
    assert evict(sinks=17) == DIM and evict(sinks=8, recent=9) == DIM
    assert evict(ws=63) == DIM and evict(tws=15) == DIM
    for more in (dict(ggml_type=0), dict(kv_heads=2), dict(head_dim=32), dict(sequences=1)):
        assert evict(to=cache(d_page_table=P + 64, d_lengths=P + 64, **more)) == DIM
    assert evict(w=None) == NULL and evict(tw=None) == NULL and evict(kept=None) == NULL


def test_softmax_and_verify_refusals():
    f = si_hip.lib().si_hip_softmax_device
    assert f(None, P, 0, 4, 1.0, P) == DIM and f(None, P, 4, 0, 1.0, P) == DIM
    assert f(None, P, 1 << 40, 1 << 30, 1.0, P) == OVER and f(None, P, 1, 1 << 31, 1.0, P) == OVER
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
        assert f(None, P, 4, 4, t, P) == RANGE
    assert f(None, P, 4, 4, 1.0, P) == NULL
    g = si_hip.lib().si_hip_verify_draft_device
    args = lambda s, m, v: (None, P, P, P, None, P, s, m, v, P, P)  # noqa: E731
    assert g(*args(0, 4, 100)) == DIM and g(*args(1, 4, 0)) == DIM
    assert g(*args(1, 0, 100)) == BATCH and g(*args(1, 17, 100)) == BATCH
    assert g(*args(1, 4, 1 << 31)) == OVER and g(*args(1 << 31, 4, 100)) == OVER
    assert g(*args(1, 4, 100)) == NULL


@pytest.mark.parametrize("n,theta,scaling", [(64, 1e7, "none"), (128, 1e4, "none"), (2, 1.0, "none"),
                                             (128, 1e6, "linear"), (128, 1e6, "yarn"),
                                             (64, 1e4, "yarn"), (256, 5e5, "yarn")])
def test_rope_frequencies(n, theta, scaling):
    code = ("none", "linear", "yarn").index(scaling)
    table, magnitude = si_hip.rope_frequencies(n, theta, code, 4.0, 32768.0)
    inv, want = R.inverse_frequencies(n, theta, scaling)
    assert table.shape == (n // 2,)
    # the f64 reference is good to about 2^-52 of the value
    assert np.allclose(table.astype(np.float64) / 2.0 ** 64 * 2 * np.pi, inv, rtol=1e-14, atol=1e-18)
    assert magnitude == pytest.approx(want, rel=1e-7)


def test_rope_frequencies_refusals():
    t, m = (C.c_uint64 * 128)(), C.c_float()
    f = si_hip.lib().si_hip_rope_frequencies
    call = lambda n=64, th=1e4, sc=0, fa=1.0, ol=1.0, bf=32.0, bs=1.0, tab=t: f(  # noqa: E731
        n, th, sc, fa, ol, bf, bs, tab, C.byref(m))
    assert call() == 0
    assert call(n=0) == DIM and call(n=63) == DIM and call(n=258) == DIM
    assert call(th=0.5) == DIM and call(th=float("nan")) == DIM and call(sc=3) == TYPE
    assert call(sc=1, fa=0.0) == DIM and call(sc=1, fa=float("inf")) == DIM
    assert call(sc=2, th=1.0) == DIM and call(sc=2, ol=0.0) == DIM and call(sc=2, bs=0.0) == DIM
    assert call(sc=2, bf=0.5) == DIM and call(tab=None) == NULL


def test_yarn_magnitude_of_a_factor_below_one():
    """The logarithm's growth is of stretched contexts; others keep their magnitude."""
    for factor, want in [(1e-6, 1.0), (0.5, 1.0), (1.0, 1.0), (1.5, 0.1 * np.log(1.5) + 1.0),
                         (40.0, 0.1 * np.log(40.0) + 1.0)]:
        _, magnitude = si_hip.rope_frequencies(64, 1e4, si_hip.ROPE_SCALING_YARN, factor, 32768.0)
        assert magnitude == pytest.approx(want, rel=1e-7)


@pytest.mark.parametrize("n,theta,scaling,factor", [
    (64, 1e7, 0, 1.0), (128, 1e6, 0, 1.0), (256, 12345.678, 0, 1.0), (128, 1e6, 1, 3.7),
    (128, 1e6, 2, 4.0), (256, 5e5, 2, 7.3), (64, 1e4, 2, 0.9)])
def test_rope_frequencies_to_the_last_bits(n, theta, scaling, factor):
    """Entries against 60 digits.  In arithmetic of 64 bits a frequency of at most a radian, 0.16
    turns, is off by some ten roundings of 2^-64, less than a unit of 2^-64 turns in all, and the
    entry's own rounding is half of one: so at most two, 2^-31 of a turn at the last position."""
    from decimal import ROUND_CEILING, ROUND_FLOOR, Decimal, localcontext
    table, _ = si_hip.rope_frequencies(n, theta, scaling, factor, 32768.0)
    with localcontext() as c:
        c.prec = 60
        pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
        log_theta, f = Decimal(theta).ln(), Decimal(factor)
        dim = lambda t: n * (Decimal(32768) / (2 * pi * t)).ln() / (2 * log_theta)  # noqa: E731
        low = max(dim(32).to_integral_value(ROUND_FLOOR), Decimal(0))
        high = min(dim(1).to_integral_value(ROUND_CEILING), Decimal(n - 1))
        for i in range(n // 2):
            inv = (-2 * Decimal(i) / n * log_theta).exp()
            if scaling == 1:
                inv /= f
            elif scaling == 2:
                ramp = min(max((i - low) / max(high - low, Decimal("0.001")), Decimal(0)), Decimal(1))
                inv = inv / f * ramp + inv * (1 - ramp)
            exact = inv / (2 * pi) * Decimal(2) ** 64
            assert abs(Decimal(int(table[i])) - exact) <= 2, i
