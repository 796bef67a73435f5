"""Layer normalisation of rows whose values add up to more than fp32 holds, or whose mean rounds by more than their deviations are."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
import test_gpu_layernorm as N  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# rows in every number of lanes and words a lane, in registers and read again
LENGTHS = [1, 5, 64, 129, 300, 1001, 2049, 5000, 9001, 20000, 40001, 70001]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
def test_equal_values(T, n, dtype):
    """Equal values have no deviations, whatever their size: y is beta, and the gradients are those of a row of zeros. The mean is off by the roundings of
    its sum, 350 of 2^-24 at most here, and the sum of what it is off by as much again: 4e-10, which is less than half a place, so the mean comes out as
    the value itself."""
    values = [1e37, -1e37, 3.3e38, -float(np.finfo(np.float32).max) if dtype == "f32" else -3.3e38, 1e30, 1.7e27, -3e22, 0.1]
    rows = len(values)
    x = L.rounded(np.repeat(np.array(values)[:, None], n, 1), dtype)
    _, gamma, beta, dy = N.case(rows, n, dtype)
    got = N.run(T, x, gamma, beta, dy, dtype)
    big = slice(0, 6)   # (beyond 1e26 squares of what the mean is off by are beyond fp32; below, they leave the variance as it comes)
    assert np.array_equal(got["mean"][big], x[big, 0])
    L.within(got["rstd"][big], np.full(6, 1 / np.sqrt(np.float64(np.float32(N.EPS)))), 4 * U / np.sqrt(N.EPS), "rstd")
    assert np.array_equal(got["y"][big], np.repeat(L.rounded(beta, dtype)[None], 6, 0))
    zero = np.zeros_like(x)
    t = N.truth(zero, gamma, beta, dy)
    b = N.bounds(zero, t, gamma, beta, dy, dtype, rows)
    L.within(got["dx"][big], t["dx"][big], b["dx"][big], "dx")
    L.within(got["dbeta"], t["dbeta"], b["dbeta"], "dbeta")
    assert np.isfinite(got["y"]).all() and np.isfinite(got["dx"]).all() and np.isfinite(got["dgamma"]).all()


@pytest.mark.parametrize("n", [2, 15, 16, 31])
def test_deviations_of_a_last_place(T, n):
    """Values of 2^85, half of them a last place, 2^62, above the others: the deviations' squares add up to less than 2^127. In last places: a value is at most 2 off the
    mean as computed, which is at most 1.6 off the true one; the sum of what it is off by goes through 10 roundings (a lane has 8 elements, then 3 steps), 16 U, of
    deviations of 0.46 and more 35 U; the variance, 0.25, is the difference of 2.6 and 2.6, 26 U and 52 U, so its root is off by 160 U at most, and y by 200 U."""
    rng = np.random.RandomState(n)
    k = np.stack([rng.permutation(np.arange(n) % 2) for _ in range(6)]).astype(np.float64)
    x = L.rounded(2.0 ** 85 + 2.0 ** 62 * k, "f32")
    d = k - k.mean(1, keepdims=True)
    want = d / np.sqrt((d * d).mean(1, keepdims=True))
    y, st = out(T, x.shape), out(T, (6, 2))
    T.layernorm_fwd(6, n, Buf(T, x), None, None, y, st, eps=N.EPS)
    L.within(y.read(), want, 200 * U * np.abs(want), "y")
    L.within(st.read()[:, 1] * 2.0 ** 62, 1 / np.sqrt((d * d).mean(1)), 165 * U / np.sqrt((d * d).mean(1)), "rstd")


def test_others_beside_them(T):
    """Rows of ordinary values, beyond fp32's sums and with NaN or infinities share workgroups; each is what it is alone."""
    for n in (20, 200):
        x, gamma, beta, dy = N.case(70, n, "f32")
        alone = N.run(T, x, gamma, beta, dy, "f32")
        x[3], x[11], x[12, 2], x[40], x[41, 0], x[69] = 2e38, -1e36, np.nan, 5e30, np.inf, 3e38
        got = N.run(T, x, gamma, beta, dy, "f32")
        same = np.setdiff1d(np.arange(70), [3, 11, 12, 40, 41, 69])
        for k in ("y", "dx", "mean", "rstd"):
            assert np.array_equal(got[k][same], alone[k][same])
        assert np.isnan(got["y"][[12, 41]]).all()
        for r in (3, 11, 40, 69):
            assert np.array_equal(got["y"][r], beta)
