"""The language-model operators at values far from one, each result held to its own size: gradients in fp16 whose dz fp16 does not
hold, and activations and their derivatives in the tails. Bounds come from the number of roundings."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ dz in fp16

def f16_bounds(x, w, z, dh):
    """(want, bound) of dx and dw under the identity as gate. dz is rounded to fp16 times a power of two that brings the
    largest into [2^14, 2^15): half a step of 2^-24 there is 2^-39 of the largest."""
    dz, dx, dw, _ = L.ff_backward(x, w, z, dh, "none")
    half = (2.0 ** -11 + 2.0 ** -22) * np.abs(dz) + 2.0 ** -39 * np.abs(dz).max()
    n, m = dz.shape

    def final(v, e):
        return e + 2.0 ** -11 * (np.abs(v) + e) + 2.0 ** -25

    size = np.abs(dz) + half
    return ((dx, final(dx, half @ np.abs(w).T + L.sum_bound(m, size @ np.abs(w).T))),
            (dw, final(dw, np.abs(x).T @ half + L.sum_bound(n, np.abs(x).T @ size))))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("size", ["large", "small", "mixed"])
@pytest.mark.parametrize("shape", [(5, 40, 24), (6, 65, 521), (40, 72, 88), (300, 333, 129), (1001, 1024, 1000), (5000, 24, 41)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_ff_gradients_whose_dz_fp16_does_not_hold(T, shape, size, accumulate):
    """dz of 10^6 beside weights of 10^-5, dz of 2^-28 beside weights of 2^13, and one sample of 10^6 among ordinary ones: dx and dw
    are well within fp16, which without a scale would have them infinite, or zero."""
    n, d, f = shape
    rng = np.random.RandomState(n + d)
    x, w, dh, z = rng.randn(n, d), rng.randn(d, 2 * f), rng.randn(n, f), rng.randn(n, 2 * f)
    if size == "large":
        x, w, dh, z = 6e-5 * x, 6e-5 * w, 1e4 * np.clip(dh, -6, 6), 100 * z
    elif size == "small":
        x, w, dh, z = 2.0 ** 13 * np.clip(x, -7, 7), 2.0 ** 13 * np.clip(w, -7, 7), 2.0 ** -8 * dh, 2.0 ** -20 * z
    else:
        x[n // 2], dh[n // 2], z[n // 2], w = 1e-4 * x[n // 2], 1e4 * np.clip(dh[n // 2], -6, 6), 100 * z[n // 2], w / 2.0 ** 14
    x, w, dh, z = (L.rounded(v, t) for v, t in ((x, "f16"), (w, "f16"), (dh, "f16"), (z, "f32")))
    bx, bw, bdh, bz = Buf(T, x, "f16"), Buf(T, w, "f16"), Buf(T, dh, "f16"), Buf(T, z)
    want = f16_bounds(x, w, z, dh)
    assert all(np.abs(v).max() < 3e4 for v, _ in want)
    before = L.rounded(rng.randn(d, 2 * f) * np.median(np.abs(want[1][0])), "f16")
    for alone in (False, True):
        dx, dw = out(T, (n, d), "f16"), Buf(T, before, "f16")
        if alone:
            T.gated_ff_bwd(d, f, False, n, bx, bw, bz, bdh, dx, None, None, act="none", dtype="f16")
            T.gated_ff_bwd(d, f, False, n, bx, bw, bz, bdh, None, dw, None, act="none", dtype="f16", accumulate=accumulate)
        else:
            T.gated_ff_bwd(d, f, False, n, bx, bw, bz, bdh, dx, dw, None, act="none", dtype="f16", accumulate=accumulate)
        L.within(dx.read(), *want[0], f"{size} dx")
        v, e = want[1]
        if accumulate:
            v, e = v + before, e + 2.0 ** -10 * (np.abs(v) + np.abs(before)) + 2.0 ** -25
        L.within(dw.read(), v, e, f"{size} dw")


def test_gated_ff_gradients_of_no_size_in_fp16(T):
    """dz of zero throughout, and infinities beside ordinary values: those stay what they are."""
    n, d, f = 9, 40, 24
    rng = np.random.RandomState(1)
    x, w, dh, z = (L.rounded(rng.randn(*s), "f16") for s in ((n, d), (d, 2 * f), (n, f), (n, 2 * f)))
    bx, bw, bz = Buf(T, x, "f16"), Buf(T, w, "f16"), Buf(T, z)
    dx, dw = out(T, (n, d), "f16"), out(T, (d, 2 * f), "f16")
    T.gated_ff_bwd(d, f, False, n, bx, bw, bz, Buf(T, 0 * dh, "f16"), dx, dw, None, act="none", dtype="f16")
    assert (dx.read() == 0).all() and (dw.read() == 0).all()
    dh[3, 5] = np.inf
    T.gated_ff_bwd(d, f, False, n, bx, bw, bz, Buf(T, dh, "f16"), dx, dw, None, act="none", dtype="f16")
    got = dx.read()
    rest = [r for r in range(n) if r != 3]
    assert not np.isfinite(got[3]).any()
    want = f16_bounds(x[rest], w, z[rest], dh[rest])[0]
    L.within(got[rest], *want, "rows beside an infinite one")
    hit = np.zeros(2 * f, bool)
    hit[[5, f + 5]] = True
    assert np.isfinite(dw.read()[:, ~hit]).all() and not np.isfinite(dw.read()[:, hit]).any()


# ------------------------------------------- activations by their own size

EPS = 2.0 ** -24   # of a rounding in fp32


def gelu_off(g):
    """What fp32 may be off: seven half-steps of each result with a reciprocal and an exponential rounded to nearest, and one
    ulp (two half-steps) more for each of the two where they are the machine's; a few for the last products."""
    from scipy.special import erfc
    cdf, pdf = 0.5 * erfc(-g / np.sqrt(2)), np.exp(-g * g / 2) / np.sqrt(2 * np.pi)
    return 16 * EPS * np.abs(g) * cdf, 16 * EPS * (cdf + np.abs(g) * pdf)


def gate(kind, g):
    """The activation and its derivative with 1 - s from an exponential, which keeps its figures in 64 bits too."""
    from scipy.special import expit
    if kind == "gelu":
        return L.gate(kind, g)
    k = 2 * np.sqrt(2 / np.pi)
    y, dy = (k * (g + 0.044715 * g ** 3), k * (1 + 3 * 0.044715 * g * g)) if kind == "gelu_tanh" else (g, 1)
    s, rest = expit(y), expit(-y)
    return (s, s * rest) if kind == "sigmoid" else (g * s, s + g * s * rest * dy)


def logistic_off(y):
    """Of 1 / (1 + exp(-y)) and of 1 minus it, relative: y's rounding and its factor's, an ulp of the exponential and the reciprocal each,
    a sum and a product."""
    return EPS * (3 * np.abs(y) + 8)


def sigmoid_off(g):
    a, slope = gate("sigmoid", g)
    return logistic_off(g) * a, 2 * (logistic_off(g) + EPS) * slope


def silu_off(g):
    s, ds = gate("sigmoid", g)
    terms = s + np.abs(g) * ds     # of s (1 + g (1 - s))
    return (logistic_off(g) + EPS) * np.abs(g) * s, (2 * logistic_off(g) + 4 * EPS) * terms


def gelu_tanh_off(g):
    from scipy.special import expit
    k = 2 * np.sqrt(2 / np.pi)
    y, dy = k * (g + 0.044715 * g ** 3), k * (1 + 3 * 0.044715 * g * g)
    s, rest = expit(y), expit(-y)
    off = EPS * (6 * np.abs(y) + 8)   # (a cube's two products and their sum more in y)
    return (off + EPS) * np.abs(g) * s, (2 * off + 8 * EPS) * (s + np.abs(g) * s * rest * dy)


# (where a result is less than 2^-126 it may be flushed)
ACT_OFF = {"gelu": (gelu_off, np.linspace(-12.5, 8, 1641)), "sigmoid": (sigmoid_off, np.linspace(-80, 80, 1601)),
           "silu": (silu_off, np.linspace(-80, 80, 1601)), "gelu_tanh": (gelu_tanh_off, np.linspace(-9.5, 9.5, 1521))}


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("n", [1, 9, 40])
@pytest.mark.parametrize("act", ACT_OFF)
def test_gated_ff_activations_by_their_own_size(T, act, n, dtype):
    """One input of 1, up columns of 1 and a gate of whatever the weight is: h is the activation itself and db, of one sample with a
    gradient, its derivative, both to be as near as their own size asks, in the tails too."""
    off, g = ACT_OFF[act]
    g = np.unique(L.rounded(g, dtype))
    f = len(g)
    z = np.tile(np.concatenate([g, np.ones(f)]), (n, 1))
    x, w = Buf(T, np.ones((n, 1)), dtype), Buf(T, z[:1], dtype)
    h, bz, db = out(T, (n, f), dtype), out(T, (n, 2 * f)), out(T, 2 * f, dtype)
    T.gated_ff_fwd(1, f, False, n, x, w, None, h, bz, act=act, dtype=dtype)
    assert np.array_equal(bz.read(), z)
    dh = Buf(T, np.eye(n)[:, :1] * np.ones((n, f)), dtype)
    T.gated_ff_bwd(1, f, True, n, x, w, bz, dh, None, None, db, act=act, dtype=dtype)
    a, slope = gate(act, g)
    a_off, slope_off = off(g)

    def final(v, e):
        return e + (0 if dtype == "f32" else L.HALF_ULP[dtype] * (np.abs(v) + e) + L.TINY[dtype])

    L.within(h.read(), np.tile(a, (n, 1)), final(a, a_off), "h")
    got = db.read()
    L.within(got[f:], a, final(a, a_off), "the up half of db")
    L.within(got[:f], slope, final(slope, slope_off), "the derivative")


# ------------------------------------------------- losses of impossible tokens

@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [9, 40, 5000])
def test_policy_loss_whose_kl_coefficient_is_zero(T, dtype, vocab):
    """A token that the model has at -inf, or 1500 below the others, beside a reference that has it: a KL term of infinity, of which a
    coefficient of 0 takes nothing. The call is the one without a reference, bit for bit."""
    rng = np.random.RandomState(vocab)
    x = L.rounded(rng.randn(5, vocab), dtype)
    x[1, 3], x[2, 3] = -np.inf, L.rounded(np.array([-1500.0]), dtype)[0]
    target, adv = np.full(5, 3, np.int32), np.ones(5)
    now = np.full(5, -2.0)
    got = []
    for ref in (None, Buf(T, now)):
        row, loss, g = out(T, 5), out(T, 1), out(T, (5, vocab), dtype)
        T.policy_loss(5, vocab, Buf(T, x, dtype), Buf(T, target, "i32"), Buf(T, now), ref, Buf(T, adv), None, None, row, loss, g, kl_coef=0.0,
                      dtype=dtype)
        got.append((row.bits(), loss.bits(), g.bits()))
        assert np.isfinite(row.read()).all() and np.isfinite(loss.read()).all() and np.isfinite(g.read()).all()
    for a, b in zip(*got):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("pairs", [1, 12])
@pytest.mark.parametrize("smoothing", [0.0, 1.0, 0.25])
@pytest.mark.parametrize("impossible", ["rejected", "chosen"])
def test_preference_loss_of_an_infinite_margin(T, impossible, smoothing, pairs):
    """An answer that the model cannot give makes its pair's margin infinite. The side that has no share in the loss adds nothing:
    without smoothing an impossible rejected answer costs nothing, and an impossible chosen one everything."""
    rows, vocab = 2 * pairs, 7
    x = np.zeros((rows, vocab))
    x[0 if impossible == "chosen" else 1, 2] = -np.inf
    start, target = np.arange(rows + 1).astype(np.int32), np.full(rows, 2, np.int32)
    margin, loss, g = out(T, pairs), out(T, 1), out(T, (rows, vocab))
    T.preference_loss(pairs, rows, vocab, Buf(T, x), Buf(T, target, "i32"), Buf(T, start, "i32"), margin=margin, loss=loss, dlogits=g,
                      beta=0.5, smoothing=smoothing)
    assert margin.read()[0] == (np.inf if impossible == "rejected" else -np.inf) and (margin.read()[1:] == 0).all()
    share = {"rejected": smoothing, "chosen": 1 - smoothing}[impossible]
    want = np.inf if share else (pairs - 1) * np.log(2.0) / pairs
    L.within(loss.read(), [want], 0 if share else 2.0 ** -23 * want)
    assert np.isfinite(g.read()).all()
