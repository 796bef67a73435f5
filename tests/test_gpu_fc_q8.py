"""Products in 8-bit integers on the GPU: the integers are exact, so a result is off by the roundings of its scaling alone."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import CANARY, Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


class Bytes:
    """int8 on the device, on a 16-byte boundary inside a larger allocation."""

    def __init__(self, T, values):
        self.shape, self.n = values.shape, values.size
        raw = np.full(256 + self.n + 256, CANARY, np.uint8)
        raw[256:256 + self.n] = np.ascontiguousarray(values, np.int8).view(np.uint8).reshape(-1)
        self.buf = T.DevBuf(raw.shape, np.uint8).upload(raw)
        self.ptr = T.DevBuf.view(self.buf.ptr.value + 256, self.shape, np.uint8).ptr

    def read(self):
        raw = self.buf.numpy()
        assert (raw[:256] == CANARY).all() and (raw[256 + self.n:] == CANARY).all(), "written outside a tensor"
        return raw[256:256 + self.n].view(np.int8).reshape(self.shape)


def quantized(x):
    """Rows in 8 bits and their scales: both quotients are fp32's."""
    x = x.astype(np.float32)
    scale = (np.abs(x).max(1) / np.float32(127)).astype(np.float32)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(scale[:, None] > 0, np.clip(np.rint(x / scale[:, None]), -127, 127), 0)
    return q.astype(np.float64), scale.astype(np.float64)


def weights(rng, n_in, n_out):
    row = (n_in + 15) // 16 * 16
    wq = np.zeros((n_out, row), np.int8)
    wq[:, :n_in] = rng.randint(-127, 128, (n_out, n_in))
    return wq, L.rounded(rng.rand(n_out) * 0.01 + 1e-4, "f32")


def truth(x, wq, ws, b):
    q, s = quantized(x)
    y = (q @ wq[:, : x.shape[1]].astype(np.float64).T) * s[:, None] * ws
    return y, np.zeros(1) if b is None else b


def bound(y, b, dtype):
    """The sum to fp32, two products with a scale and the bias: four roundings, and the result's."""
    e = 2.0 ** -24 * 4 * (np.abs(y) + np.abs(b))
    return e + L.HALF_ULP[dtype] * (np.abs(y + b) + e) + L.TINY[dtype]


# a few samples and many, every tile, sums split and whole, odd ends; sums beyond 2^24; a row that is one byte
SHAPES = [(1, 1, 1), (1, 4096, 40), (2, 17, 3), (3, 1000, 130), (4, 257, 1000), (5, 2048, 64), (8, 64, 513), (8, 6160, 33), (1, 50000, 20), (9, 64, 16),
          (16, 4096, 100), (20, 33, 700), (33, 515, 1300), (64, 2000, 260), (77, 1001, 2731), (130, 128, 130), (200, 16, 4000), (300, 700, 513),
          (1000, 96, 1030), (1500, 1024, 1025), (3, 131072, 5), (12, 100000, 40)]


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_forward(T, shape, dtype, bias):
    n, d, f = shape
    rng = np.random.RandomState(n + 3 * d + 7 * f)
    x = L.rounded(rng.randn(n, d) * np.exp(rng.randn(n, 1)), dtype)
    wq, ws = weights(rng, d, f)
    b = L.rounded(rng.randn(f), dtype) if bias else None
    skew = 1 if d % 2 or f % 2 else 0
    y = out(T, (n, f), dtype, skew)
    T.fc_q8_fwd(d, f, bias, n, Buf(T, x, dtype, skew), Bytes(T, wq), Buf(T, ws), Buf(T, b, dtype, skew) if bias else None, y, dtype=dtype)
    want, shift = truth(x, wq, ws, b)
    L.within(y.read(), want + shift, bound(want, shift, dtype), f"{shape} {dtype}")


@pytest.mark.parametrize("n", [1, 3, 40])
def test_the_integers_are_exact(T, n):
    """Whole numbers with a largest size of 127 are their own 8-bit form, and a scale of one leaves the sums: each is a whole number below 2^24."""
    rng = np.random.RandomState(n)
    d, f = 1000, 300
    x = rng.randint(-127, 128, (n, d)).astype(np.float64)
    x[:, 0] = 127
    wq, _ = weights(rng, d, f)
    y = out(T, (n, f))
    T.fc_q8_fwd(d, f, False, n, Buf(T, x), Bytes(T, wq), Buf(T, np.ones(f)), None, y)
    assert np.array_equal(y.read(), x @ wq[:, :d].T.astype(np.float64))


@pytest.mark.parametrize("n", [2, 30])
def test_ties_and_exceptional_samples(T, n):
    d, f = 130, 20
    rng = np.random.RandomState(1)
    x = rng.randn(n, d)
    x[0] = 0.0                                  # gives the bias
    x[1] = (rng.randint(-126, 127, d) + 0.5)    # halves: to the even neighbour
    x[1, 3] = 127.0
    if n > 2:
        x[2, 5], x[3, 6], x[4, 7] = np.nan, np.inf, -np.inf
        x[5] *= 1e-42                           # a scale among fp32's smallest
        x[6] *= 3e37
        x[7], x[7, 9] = 0.0, -5.0
    x = L.rounded(x, "f32")
    wq, ws = weights(rng, d, f)
    b = L.rounded(rng.randn(f), "f32")
    y = out(T, (n, f))
    T.fc_q8_fwd(d, f, True, n, Buf(T, x), Bytes(T, wq), Buf(T, ws), Buf(T, b), y)
    got = y.read()
    bad = [] if n == 2 else [2, 3, 4]
    assert np.isnan(got[bad]).all()
    fine = [i for i in range(n) if i not in bad]
    want, _ = truth(x[fine], wq, ws, b)
    L.within(got[fine], want + b, bound(want, b, "f32") + 2.0 ** -149, "fine rows")
    assert np.array_equal(got[0], b)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (5, 64), (64, 65), (130, 17), (1000, 300), (2049, 100)])
def test_pack(T, shape, dtype):
    d, f = shape
    rng = np.random.RandomState(d)
    w = L.rounded(rng.randn(d, f) / np.sqrt(d), dtype)
    w[:, 0] = 0.0
    row = T.q8_row(d)
    assert row == (d + 15) // 16 * 16
    wq, ws = Bytes(T, np.full((f, row), 3, np.int8)), out(T, f)
    T.fc_q8_pack(d, f, Buf(T, w, dtype), wq, ws, dtype=dtype)
    q, s = quantized(w.T)
    assert np.array_equal(ws.read(), s) and np.array_equal(wq.read()[:, :d], q) and (wq.read()[:, d:] == 0).all()
    # and the two together are near the layer in floating point: a rounding of half a step of 127 of the largest on either side
    x = L.rounded(rng.randn(12, d), dtype)
    y = out(T, (12, f), dtype)
    T.fc_q8_fwd(d, f, False, 12, Buf(T, x, dtype), wq, ws, None, y, dtype=dtype)
    sx, sw = np.abs(x).max(1)[:, None] / 254 * 1.001, np.abs(w).max(0) / 254 * 1.001
    e = sx * np.abs(w).sum(0) + np.abs(x).sum(1)[:, None] * sw + d * sx * sw
    L.within(y.read(), x @ w, e + L.HALF_ULP[dtype] * (np.abs(x @ w) + e) + L.TINY[dtype], "the layer")


def test_pack_of_exceptional_weights(T):
    w = np.ones((40, 4))
    w[3, 1], w[5, 2] = np.nan, np.inf
    wq, ws = Bytes(T, np.full((4, 48), 3, np.int8)), out(T, 4)
    T.fc_q8_pack(40, 4, Buf(T, w), wq, ws)
    assert np.isnan(ws.read()[1:3]).all() and np.isfinite(ws.read()[[0, 3]]).all()
    y = out(T, (2, 4))
    T.fc_q8_fwd(40, 4, False, 2, Buf(T, np.ones((2, 40))), wq, ws, None, y)
    assert np.isnan(y.read()[:, 1:3]).all() and np.isfinite(y.read()[:, [0, 3]]).all()


def test_no_samples(T):
    b = Buf(T, np.ones(4))
    T.fc_q8_fwd(40, 4, False, 0, b, b, b, None, b)
