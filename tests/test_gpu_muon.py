"""The orthogonalised update on the GPU against its definition in 64 bits. The bound of one step is worked out element by element from the roundings of
operands and sums; later steps add their own to what the earlier ones grew to."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu

A, B, C, EPS = 3.4445, -4.7750, 2.0315, 1e-7
U = 2.0 ** -24


def f32(v):
    return float(np.float32(v))


a, b, c = f32(A), f32(B), f32(C)


def step(x, co=(a, b, c)):
    if x.shape[0] > x.shape[1]:
        return step(x.T, co).T
    g = x @ x.T
    return co[0] * x + (co[1] * g + co[2] * g @ g) @ x


def start(u, eps=f32(EPS)):
    return u / (np.sqrt((u * u).sum()) + eps)


# of an operand: hi alone is off by half a step of fp16 (2^-11), hi + lo by that of lo, and the product of the two los is left out
OPERAND = {"f16": 2.0 ** -11, "f32": 2.0 ** -22}
FLOOR = 2.0 ** -25      # half of fp16's smallest step, of what is held around 2^14 and more times its size


def sum_error(k):
    """Of a sum of k products, by the sum of their sizes: the additions of the parts and the matrix instruction's truncations, 16 at a time."""
    return (k / 8 + 40) * 2.0 ** -23


def step_bound(x, products, flat):
    """How far one step of x may be from step(x), element by element. flat: what the diagonal of the Gram matrix is relieved of."""
    if x.shape[0] > x.shape[1]:
        return step_bound(x.T, products, flat).T
    e = OPERAND[products]
    m, n = x.shape
    ax = np.abs(x)
    ex = e * ax + FLOOR * 2.0 ** -12
    g = x @ x.T - flat * np.eye(m)
    ag = np.abs(g)
    full = ax @ ax.T
    eg = ax @ ex.T + ex @ ax.T + sum_error(n) * full + U * (full + flat)
    eg = eg + e * (ag + eg) + FLOOR * 2.0 ** -12
    one, beta = abs(b + 2 * c * flat), abs(a + b * flat + c * flat * flat)
    p = np.abs((b + 2 * c * flat) * g + c * g @ g)
    ep = one * eg + c * (ag @ eg + eg @ ag + sum_error(m) * ag @ ag) + 4 * U * (one * ag + c * ag @ ag)
    ep = ep + e * (p + ep) + FLOOR * 2.0 ** -12
    return ep @ ax + p @ ex + (sum_error(m) + 4 * U) * p @ ax + beta * (2.0 ** -22 * ax + FLOOR * 2.0 ** -12) + 4 * U * beta * ax


def matrix(rows, cols, dtype, kind="gauss"):
    rng = np.random.RandomState(rows * 7 + cols)
    u = rng.randn(rows, cols)
    if kind == "falling":   # some strong directions of falling strength, as gradients have
        k = min(rows, cols, 16)
        u = 3 * (rng.randn(rows, k) * np.logspace(0, -2, k)) @ rng.randn(k, cols) + 0.3 * u
    return L.rounded(1e-3 * u, dtype)


SHAPES = [(1, 1), (1, 9), (9, 1), (3, 5), (17, 17), (64, 64), (65, 33), (40, 100), (120, 84), (130, 257), (300, 129), (257, 640), (513, 200),
          (520, 520), (1000, 65)]


@pytest.mark.parametrize("products", ["f32", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", L.DTYPES)
def test_one_step(T, shape, dtype, products):
    u = matrix(*shape, dtype)
    skew = 1 if shape[1] % 2 else 0
    bu, y = Buf(T, u, dtype, skew), out(T, shape, dtype, skew)
    T.orthogonalize(T.muon_desc(steps=1, products=products), *shape, bu, y, dtype=dtype)
    x = start(u)
    want, e = step(x), step_bound(x, products, 1.0 / min(shape))
    e = e + 4 * U * np.abs(want) + 12 * U * np.abs(x)   # (the start's own rounding, which a step makes 4 times as large at most)
    L.within(y.read(), want, e + L.HALF_ULP[dtype] * (np.abs(want) + e) + L.TINY[dtype], f"{shape} {dtype} {products}")
    T.orthogonalize(T.muon_desc(steps=1, products=products), *shape, bu, bu, dtype=dtype)   # in place
    assert np.array_equal(bu.bits(), y.bits())


@pytest.mark.parametrize("shape", [(700, 900), (1030, 300), (260, 2100), (2000, 1999)])
@pytest.mark.parametrize("products", ["f32", "f16"])
def test_one_step_of_large_matrices(T, shape, products):
    """Every tile shape, several tiles along either side and a last one that is not full."""
    u = matrix(*shape, "f32")
    bu, y = Buf(T, u), out(T, shape)
    T.orthogonalize(T.muon_desc(steps=1, products=products), *shape, bu, y)
    x = start(u)
    want, e = step(x), step_bound(x, products, 1.0 / min(shape)) + 12 * U * np.abs(x)
    L.within(y.read(), want, e + 5 * U * np.abs(want), f"{shape} {products}")


@pytest.mark.parametrize("shape", [(1, 1), (37, 37), (120, 84), (84, 520), (600, 400)])
@pytest.mark.parametrize("kind", ["gauss", "falling"])
@pytest.mark.parametrize("steps", [2, 5, 6])
def test_steps(T, shape, kind, steps):
    """A step takes an error to 4 times its size at most: the slope of a s + b s^3 + c s^5 is below 4 for all s up to 1.21, the largest that it gives."""
    u = matrix(*shape, "f32", kind)
    x, e = start(u), 0.0
    e = 12 * U * np.linalg.norm(x)
    flat = 1.0 / min(shape)
    for _ in range(steps):
        e = 4 * e + np.linalg.norm(step_bound(x, "f32", flat))
        x = step(x)
        s = np.sqrt(flat)
        flat = (s * (a + b * flat + c * flat * flat)) ** 2
    bu, y = Buf(T, u), out(T, shape)
    T.orthogonalize(T.muon_desc(steps=steps), *shape, bu, y)
    assert np.linalg.norm(y.read() - x) <= e + U * np.linalg.norm(x)
    # operands in fp16: four times what the interface says
    T.orthogonalize(T.muon_desc(steps=steps, products="f16"), *shape, bu, y)
    assert np.linalg.norm(y.read() - x) <= 4e-3 * np.linalg.norm(x)


def test_singular_values(T):
    """Singular vectors stay, and a singular value s of the start becomes a s + b s^3 + c s^5, again and again."""
    rng = np.random.RandomState(3)
    q1, _ = np.linalg.qr(rng.randn(96, 96))
    q2, _ = np.linalg.qr(rng.randn(200, 96))
    s = np.linspace(0.02, 1.0, 96)
    s /= np.sqrt((s * s).sum())
    u = L.rounded(q1 @ np.diag(s) @ q2.T * 40, "f32")
    y = out(T, u.shape)
    T.orthogonalize(T.muon_desc(), *u.shape, Buf(T, u), y)
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    got = y.read()
    assert np.abs(q1.T @ got @ q2 - np.diag(s)).max() < 1e-4
    assert np.abs(np.sort(np.linalg.svd(got)[1]) - np.sort(s)).max() < 1e-4


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("nesterov", [True, False])
def test_update(T, dtype, nesterov):
    shape = (90, 130)
    rng = np.random.RandomState(8)
    w, mom = L.rounded(rng.randn(*shape) * 0.1, "f32"), L.rounded(1e-2 * rng.randn(*shape), "f32")
    bw, bm = Buf(T, w), Buf(T, mom)
    alpha, mu, lam, scale, gs = (f32(v) for v in (0.05, 0.9, 0.1, 1.25, 0.5))
    o = T.muon_desc(alpha=alpha, mu=mu, lambda_=lam, scale=scale, nesterov=nesterov, steps=5)
    for turn in range(3):
        g = matrix(shape[0], shape[1] , dtype) * (turn + 1)
        g = L.rounded(g, dtype)
        T.muon_update(o, *shape, Buf(T, g, dtype), bw, bm, grad_scale=gs, dtype=dtype)
        mom = mu * mom + g * gs
        L.within(bm.read(), mom, 3 * (turn + 1) * U * (np.abs(mom) + np.abs(g)), "momentum")
        x = start(g * gs + mu * mom if nesterov else mom)
        e, flat = 40 * U * np.linalg.norm(x), 1.0 / 90
        for _ in range(5):
            e = 4 * e + np.linalg.norm(step_bound(x, "f32", flat))
            x = step(x)
            s = np.sqrt(flat)
            flat = (s * (a + b * flat + c * flat * flat)) ** 2
        w = w - alpha * (scale * x + lam * w)
        got = bw.read()
        assert np.linalg.norm(got - w) <= alpha * scale * e + 8 * U * np.linalg.norm(w)
        w, mom = got, bm.read()


def test_without_steps_and_zero_and_scale(T):
    u = matrix(33, 70, "f32")
    y = out(T, u.shape)
    T.orthogonalize(T.muon_desc(steps=0), 33, 70, Buf(T, u), y)
    x = start(u)
    L.within(y.read(), x, 2.0 ** -22 * np.abs(x) + FLOOR * 2.0 ** -12, "no steps")
    T.orthogonalize(T.muon_desc(), 33, 70, Buf(T, 0 * u), y)
    assert (y.read() == 0).all()
    want = out(T, u.shape)
    T.orthogonalize(T.muon_desc(eps=1e-30), 33, 70, Buf(T, u), want)
    for f in (2.0 ** 100, 2.0 ** -60):   # the size of U does not matter
        T.orthogonalize(T.muon_desc(eps=1e-30), 33, 70, Buf(T, L.rounded(u * f, "f32")), y)
        L.within(y.read(), want.read(), 2.0 ** -20 * np.abs(want.read()) + 1e-6, "scaled")
    u[3, 4] = np.nan
    T.orthogonalize(T.muon_desc(), 33, 70, Buf(T, u), y)
    assert np.isnan(y.read()).all()
    for shape in ((0, 5), (5, 0)):
        T.orthogonalize(T.muon_desc(), *shape, y, y)


def test_other_coefficients(T):
    u = matrix(50, 80, "f32")
    y = out(T, u.shape)
    T.orthogonalize(T.muon_desc(a=1.5, b=-0.5, c=0.0, steps=12), 50, 80, Buf(T, u), y)   # the cubic, which converges to one
    x = start(u)
    for _ in range(12):
        x = step(x, (1.5, -0.5, 0.0))
    # slope 1.5 at most, 12 steps of less than 2^-19 of X each
    assert np.linalg.norm(y.read() - x) <= 1.5 ** 12 * 2 * 2.0 ** -19 * np.linalg.norm(x)


def test_same_bits_again(T):
    u = matrix(300, 500, "bf16")
    y, z = out(T, u.shape, "bf16"), out(T, u.shape, "bf16")
    for p in ("f32", "f16"):
        T.orthogonalize(T.muon_desc(products=p), 300, 500, Buf(T, u, "bf16"), y, dtype="bf16")
        T.orthogonalize(T.muon_desc(products=p), 300, 500, Buf(T, u, "bf16"), z, dtype="bf16")
        assert np.array_equal(y.bits(), z.bits())


@pytest.mark.parametrize("shape", [(1, 20000), (20001, 1), (2, 17001), (9003, 7), (31, 900), (1031, 33), (5, 70001)])
@pytest.mark.parametrize("products", ["f32", "f16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_step_of_long_thin_matrices(T, shape, products, dtype):
    u = matrix(*shape, dtype)
    bu, y = Buf(T, u, dtype, shape[1] % 2), out(T, shape, dtype, shape[1] % 2)
    T.orthogonalize(T.muon_desc(steps=1, products=products), *shape, bu, y, dtype=dtype)
    x = start(u)
    want, e = step(x), step_bound(x, products, 1.0 / min(shape)) + 12 * U * np.abs(x)
    e = e + 5 * U * np.abs(want)
    L.within(y.read(), want, e + L.HALF_ULP[dtype] * (np.abs(want) + e) + L.TINY[dtype], f"{shape} {dtype} {products}")


def test_many_steps_and_every_coefficient(T):
    """32 steps, and coefficients whose largest polynomial or singular value lies inside the range rather than at its end."""
    u = matrix(70, 300, "f32")
    y = out(T, u.shape)
    for co, steps in (((1.5, -0.5, 0.0), 32), ((1.875, -1.25, 0.375), 20), ((1.0, 0.0, 0.0), 7), ((2.0, -1.5, 0.5), 10), ((0.5, 0.25, 0.0), 9)):
        T.orthogonalize(T.muon_desc(steps=steps, **dict(zip("abc", co))), 70, 300, Buf(T, u), y)
        x, slope = start(u), 1.0
        e = 12 * U * np.linalg.norm(x)
        for _ in range(steps):
            s = np.linspace(0, max(1.0, np.linalg.svd(x)[1][0]), 200)
            slope = max(1.0, np.abs(co[0] + 3 * co[1] * s ** 2 + 5 * co[2] * s ** 4).max())
            # a step's own: the operands' 2^-22, of X and of two Gram matrices, and the sums' of up to 300 products
            e = slope * e + (8 * 2.0 ** -22 + 3 * sum_error(300)) * (abs(co[0]) + abs(co[1]) + abs(co[2])) * np.linalg.norm(x)
            x = step(x, co)
        assert np.linalg.norm(y.read() - x) <= e + U * np.linalg.norm(x), co
