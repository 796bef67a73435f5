"""The language-model operators at the sizes where another kernel takes over, and at their limits, against the definitions in 64 bits."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


def whole_numbers(rng, shape, most):
    """Whole numbers, so few that sums of their products are exact in fp32: one term lost or taken twice shows."""
    return rng.randint(-most, most + 1, shape).astype(np.float64)


def ff_exact_case(T, shape, dtype, bias=False, accumulate=False, skew=0, most=2, seed=0):
    """The block with the identity as its gate on whole numbers: z and dz are whole numbers and every sum of products below
    2^24, so that z, and in fp32 every result, has to be equal; in 16 bits results are the sums rounded once."""
    n, d, f = shape
    rng = np.random.RandomState(seed + n + d + f)
    # (sparse: the sums of products stay small)
    x, w, b, dh = (whole_numbers(rng, s, most) * (rng.rand(*s) < 0.3) for s in ((n, d), (d, 2 * f), (2 * f,), (n, f)))
    b = b if bias else None
    z = x @ w + (0 if b is None else b)
    limit = {"f32": 2 ** 24, "bf16": 2 ** 8, "f16": 2 ** 11}[dtype]
    zk = np.clip(np.round(z), -2, 2)      # what the backward pass is given: any z
    dz, dx, dw, db = L.ff_backward(x, w, zk, dh, "none")
    sizes = np.abs(x) @ np.abs(w) + (0 if b is None else np.abs(b)), np.abs(dz) @ np.abs(w).T, np.abs(x).T @ np.abs(dz), np.abs(dz).sum(0)
    assert np.abs(dz).max() <= limit and max(v.max() for v in sizes) < 2 ** 24
    bx, bw, bdh = (Buf(T, v, dtype, skew) for v in (x, w, dh))
    bb = Buf(T, b, dtype, skew) if bias else None
    h, bz = out(T, (n, f), dtype, skew), out(T, (n, 2 * f), "f32", skew)
    T.gated_ff_fwd(d, f, bias, n, bx, bw, bb, h, bz, act="none", dtype=dtype)
    what = f"{dtype} batch {n} {d}->2*{f} skew {skew}"
    assert np.array_equal(bz.read(), z), what + " z"
    prod = z[:, :f] * z[:, f:]
    exact = np.abs(prod) < 2 ** 24
    L.within(h.read(), np.where(exact, L.rounded(prod, dtype), prod), np.where(exact, 0, (2.0 ** -23 + L.HALF_ULP[dtype]) * np.abs(prod)), what + " h")
    before = [whole_numbers(rng, s, 3) for s in ((d, 2 * f), (2 * f,))]
    bdx, bdw = out(T, (n, d), dtype, skew), Buf(T, before[0], dtype, skew)
    bdb = Buf(T, before[1], dtype, skew) if bias else None
    T.gated_ff_bwd(d, f, bias, n, bx, bw, Buf(T, zk, "f32", skew), bdh, bdx, bdw, bdb, act="none", dtype=dtype, accumulate=accumulate)
    add = 1 if accumulate else 0
    for got, want, name in ((bdx, dx, "dx"), (bdw, dw + add * before[0], "dw"), (bdb, db + add * before[1], "db")):
        if got is not None:
            L.within(got.read(), L.rounded(want, dtype), 0.0, what + " " + name)


@pytest.mark.parametrize("n", [5, 8])
@pytest.mark.parametrize("f", [1, 3])
def test_gated_ff_of_the_most_inputs(T, n, f):
    """(fp32: the weight gradient's tiles of rows, of which a launch takes 65535)"""
    ff_exact_case(T, (n, (1 << 21) - 1, f), "f32", bias=True)
