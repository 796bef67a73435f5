"""Layer normalisation on the GPU against its definition in 64 bits, at every way a row can lie in lanes and workgroups. Bounds come from
the number of roundings."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = 2.0 ** -24


def truth(x, gamma, beta, dy, eps=EPS):
    n = x.shape[1]
    mean = x.mean(1, keepdims=True)
    d = x - mean
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    xhat = d * rstd
    g = dy * gamma
    c1, c2 = g.mean(1, keepdims=True), (g * xhat).mean(1, keepdims=True)
    return {"mean": mean[:, 0], "rstd": rstd[:, 0], "y": xhat * gamma + beta, "dx": rstd * (g - c1 - xhat * c2),
            "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0), "xhat": xhat, "g": g, "c1": c1, "c2": c2, "n": n}


def depth(n):
    """Roundings that a sum of n terms goes through: a lane has 128 at most (of longer rows n / 1024), then 6 steps of a wave, 16 waves."""
    return max(128, n // 1024 * 8 + 8) + 6 + 16


def bounds(x, t, gamma, beta, dy, dtype, rows_sum):
    """What fp32 sums and one rounding of each result may add up to. A deviation x - mean rounds, unless the two are within a factor of two of
    each other (then it is exact, but as far off as the mean, k of it), and what is off in all of a row's deviations is taken off again, but for the
    rounding of their sum; rstd is off by half of the variance's relative error."""
    k = depth(t["n"]) * U
    h, tiny = L.HALF_ULP[dtype], L.TINY[dtype]
    mean = np.abs(t["mean"])[:, None]
    size = np.abs(x - t["mean"][:, None]).mean(1, keepdims=True) + k * np.abs(x).mean(1, keepdims=True)
    near = np.abs(x - t["mean"][:, None]) < 0.4 * mean
    dev = np.where(near, 0, U * (np.abs(x) + mean)) + 4 * U * np.abs(x - t["mean"][:, None]) + 4 * k * size   # of x - mean
    rel = 2 * k + 8 * U + 2 * (dev * t["rstd"][:, None]).max(1, keepdims=True)              # of rstd
    xh = dev * t["rstd"][:, None] + (rel + 4 * U) * np.abs(t["xhat"])
    g, c1, c2, xhat = t["g"], t["c1"], t["c2"], t["xhat"]
    ag, ax = np.abs(g), np.abs(xhat)
    e1 = 2 * k * ag.mean(1, keepdims=True)
    e2 = 2 * k * (ag * (ax + 1)).mean(1, keepdims=True) + (ag * xh).mean(1, keepdims=True) + np.abs(c2) * rel
    inner = 2 * U * ag + e1 + e2 * ax + np.abs(c2) * xh + 4 * U * (ag + np.abs(c1) + ax * np.abs(c2))
    edx = t["rstd"][:, None] * (inner * (1 + rel) + rel * (ag + np.abs(c1) + ax * np.abs(c2)))
    ey = np.abs(gamma) * xh + 2 * U * (np.abs(gamma) * ax + np.abs(beta))
    s = (rows_sum + 64) * U
    eg = (np.abs(dy) * xh).sum(0) + s * (np.abs(dy) * (ax + xh)).sum(0)
    eb = s * np.abs(dy).sum(0)

    def final(v, e):
        return e + h * (np.abs(v) + e) + tiny

    return {"mean": dev.max(1) + U * np.abs(t["mean"]), "rstd": t["rstd"] * (rel[:, 0] + 4 * U), "y": final(t["y"], ey),
            "dx": final(t["dx"], edx), "dgamma": final(t["dgamma"], eg), "dbeta": final(t["dbeta"], eb)}


def case(rows, n, dtype, seed=0, offset=0.0):
    rng = np.random.RandomState(seed + 31 * rows + n)
    x = L.rounded(rng.randn(rows, n) * 1.5 + offset + rng.randn(rows, 1), dtype)
    return x, L.rounded(1 + 0.2 * rng.randn(n), dtype), L.rounded(0.3 * rng.randn(n), dtype), L.rounded(rng.randn(rows, n), dtype)


def run(T, x, gamma, beta, dy, dtype, skew=0, eps=EPS):
    rows, n = x.shape
    bx, bg, bb, bd = (None if v is None else Buf(T, v, dtype, skew) for v in (x, gamma, beta, dy))
    y, dx, dg, db = (out(T, s, dtype, skew) for s in ((rows, n), (rows, n), (n,), (n,)))
    st = out(T, (rows, 2))
    T.layernorm_fwd(rows, n, bx, bg, bb, y, st, eps=eps, dtype=dtype)
    T.layernorm_bwd(rows, n, bx, bg, st, bd, dx, dg, db, dtype=dtype)
    s = st.read()
    return {"y": y.read(), "dx": dx.read(), "dgamma": dg.read(), "dbeta": db.read(), "mean": s[:, 0], "rstd": s[:, 1]}


# every split of a row over lanes: 8, 32, 64 (1, 2, 4, 8 words), 256, 512 and 1024 of them, rows that no registers hold, at odd ends
SHAPES = [(1, 1), (3, 2), (1, 7), (130, 64), (37, 65), (5, 256), (600, 100), (33, 257), (9, 1000), (1030, 520), (1100, 1025), (1029, 2047),
          (6, 2049), (1025, 4096), (3, 4097), (5, 8192), (2, 8193), (3, 16385), (9, 20001), (2, 70001), (17, 9000)]


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(T, shape, dtype):
    x, gamma, beta, dy = case(*shape, dtype)
    t = truth(x, gamma, beta, dy)
    b = bounds(x, t, gamma, beta, dy, dtype, shape[0])
    got = run(T, x, gamma, beta, dy, dtype, skew=1 if shape[1] % 2 else 0)
    for k in b:
        L.within(got[k], t[k], b[k], f"{k} {shape} {dtype}")


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_without_gamma_and_beta(T, dtype):
    x, _, _, dy = case(11, 300, dtype)
    t = truth(x, np.ones(300), np.zeros(300), dy)
    got = run(T, x, None, None, dy, dtype)
    b = bounds(x, t, np.ones(300), np.zeros(300), dy, dtype, 11)
    for k in b:
        L.within(got[k], t[k], b[k], k)


@pytest.mark.parametrize("shape", [(19, 333), (3, 9001)])
def test_rows_far_from_zero(T, shape):
    """The deviations keep their figures where the mean is 10^4 times as large."""
    x, gamma, beta, dy = case(*shape, "f32", offset=1e4)
    t = truth(x, gamma, beta, dy)
    got = run(T, x, gamma, beta, dy, "f32")
    b = bounds(x, t, gamma, beta, dy, "f32", shape[0])
    for k in b:
        L.within(got[k], t[k], b[k], k)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", [(5, 12), (40, 700), (3, 9001)])
def test_strides_in_place_and_parts(T, shape, dtype):
    rows, n = shape
    x, gamma, beta, dy = case(rows, n, dtype)
    base = run(T, x, gamma, beta, dy, dtype)
    ld = n + 13
    wide = lambda v: np.concatenate([v, np.full((rows, 13), 9.0)], 1)  # noqa: E731
    bx, bd, bg, bb = Buf(T, wide(x), dtype), Buf(T, wide(dy), dtype), Buf(T, gamma, dtype), Buf(T, beta, dtype)
    y, st, dg, db = out(T, (rows, ld), dtype), out(T, (rows, 2)), Buf(T, np.ones(n), dtype), Buf(T, np.ones(n), dtype)
    T.layernorm_fwd(rows, n, bx, bg, bb, y, st, eps=EPS, dtype=dtype, ld=ld, ld_y=ld)
    assert np.array_equal(y.read()[:, :n], base["y"]) and (y.read()[:, n:] == 3.25).all()
    only = out(T, (n,), dtype)
    T.layernorm_bwd(rows, n, bx, bg, st, bd, None, only, None, dtype=dtype, ld=ld, ld_dy=ld)   # one of the three alone
    assert np.array_equal(only.read(), base["dgamma"])
    T.layernorm_bwd(rows, n, bx, bg, st, bd, None, None, only, dtype=dtype, ld=ld, ld_dy=ld)
    assert np.array_equal(only.read(), base["dbeta"])
    T.layernorm_bwd(rows, n, bx, bg, st, bd, bd, dg, db, dtype=dtype, ld=ld, ld_dy=ld, ld_dx=ld, accumulate=True)   # over dy
    assert np.array_equal(bd.read()[:, :n], base["dx"]) and (bd.read()[:, n:] == 9.0).all()
    t = truth(x, gamma, beta, dy)
    b = bounds(x, t, gamma, beta, dy, dtype, rows)
    for k, v in (("dgamma", dg), ("dbeta", db)):
        L.within(v.read(), t[k] + 1, b[k] + (L.HALF_ULP[dtype] + U) * (1 + np.abs(t[k] + 1)), k + " added")
    T.layernorm_fwd(rows, n, bx, bg, bb, bx, st, eps=EPS, dtype=dtype, ld=ld, ld_y=ld)   # over x
    assert np.array_equal(bx.read()[:, :n], base["y"]) and (bx.read()[:, n:] == 9.0).all()


@pytest.mark.parametrize("n", [5, 700, 3000, 9001])
def test_exceptional_rows(T, n):
    """A row of equal values gives beta; a NaN or an infinity stays in its own row and in the gradients that add it up."""
    x, gamma, beta, dy = case(6, n, "f32")
    x[1] = 12345.678
    x[3, n // 2] = np.nan
    x[4, 0] = np.inf
    got = run(T, x, gamma, beta, dy, "f32")
    x32 = np.float64(np.float32(12345.678))
    L.within(got["y"][1], beta, 4 * (depth(n) * U) ** 2 * x32 / np.sqrt(EPS) * np.abs(gamma) + 2 * U * np.abs(beta), "equal values")
    assert np.isnan(got["y"][3]).all() and np.isnan(got["y"][4]).all() and np.isnan(got["dx"][3:5]).all()
    assert np.isnan(got["dgamma"]).all() and np.isfinite(got["dbeta"]).all()
    fine = [0, 2, 5]
    t = truth(x[fine], gamma, beta, dy[fine])
    b = bounds(x[fine], t, gamma, beta, dy[fine], "f32", 3)
    for k in ("y", "dx", "mean", "rstd"):
        L.within(got[k][fine], t[k], b[k], k)


def test_no_rows(T):
    one, n = Buf(T, np.ones(9), "f16"), 9
    dg, db = out(T, n, "f16", 1), out(T, n, "f16", 1)
    T.layernorm_fwd(0, n, one, None, None, one, None, dtype="f16")
    T.layernorm_bwd(0, n, one, None, None, one, None, dg, db, dtype="f16", accumulate=True)
    assert (dg.read() == 3.25).all()
    T.layernorm_bwd(0, n, one, None, None, one, None, dg, db, dtype="f16")
    assert (dg.read() == 0).all() and (db.read() == 0).all()


def test_gradients_against_differences(T):
    """A loss sum(y c) by central differences of the forward pass."""
    rows, n = 3, 10
    x, gamma, beta, c = case(rows, n, "f32")
    got = run(T, x, gamma, beta, c, "f32")
    bx, y = None, out(T, (rows, n))

    def loss(x, gamma, beta):
        bx, bg, bb = Buf(T, x), Buf(T, gamma), Buf(T, beta)
        T.layernorm_fwd(rows, n, bx, bg, bb, y, None, eps=EPS)
        return (y.read() * c).sum()

    h = 2.0 ** -7
    for what, arrays, grad in (("dx", 0, got["dx"]), ("dgamma", 1, got["dgamma"]), ("dbeta", 2, got["dbeta"])):
        args = [x, gamma, beta]
        diff = np.zeros_like(args[arrays])
        for i in np.ndindex(diff.shape):
            v = []
            for s in (h, -h):
                a = [q.copy() for q in args]
                a[arrays][i] += s
                v.append(loss(*a))
            diff[i] = (v[0] - v[1]) / (2 * h)
        # a difference is off by h^2 / 6 of the third derivative (below 40 here: deviations of 1.5, a spread of one) and the outputs' roundings
        L.within(grad, diff, 40 * h * h / 6 + 16 * U * np.abs(c).sum() * 4 / h, what)


def test_same_bits_again(T):
    x, gamma, beta, dy = case(3000, 520, "bf16")
    a, b = run(T, x, gamma, beta, dy, "bf16"), run(T, x, gamma, beta, dy, "bf16")
    assert all(np.array_equal(a[k], b[k]) for k in a)
