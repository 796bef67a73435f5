"""The gradients of gamma and beta where every workgroup goes through a long series of rows, as near to 64 bits as the depth of the kernels' sums makes them."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
import test_gpu_layernorm as N  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def lanes_of(n):
    return 8 if n <= 64 else 32 if n <= 256 else 64 if n <= 1024 else 128 if n <= 2048 else 256 if n <= 4096 else 512


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("rows,n", [(200001, 24), (100003, 3), (40009, 200), (12007, 700), (6011, 1500), (2777, 3001), (1999, 5003), (900, 9001), (4099, 8200)])
def test_gradients_of_many_rows(T, rows, n, dtype):
    """A thread adds up its rows one after the other, then the lanes that have the same columns (3 steps at most) and the sets in LDS (8 at most), then the workgroups'
    sums: 256 at most in groups of 32, and the 32 groups. Long rows: bands of rows, 256 compute units times 8 by the columns' strips of 1024, or of eight rows."""
    cus = T.device_info()[1]
    if n <= 8192:
        at_a_time = 512 // lanes_of(n)
        parts = min(-(-rows // at_a_time), cus)
        serial = -(-rows // (parts * at_a_time)) + 3 + 8
    else:
        band = max(8, -(-rows // max(1, 8 * cus // -(-n // 1024))))
        parts, serial = -(-rows // band), band
    depth = serial + -(-parts // 32) + 32
    x, gamma, beta, dy = N.case(rows, n, dtype)
    t = N.truth(x, gamma, beta, dy)
    # of a row: what its mean and its spread are off by, from sums that a lane begins with 64 elements at most, in 6 steps of a wave and 16 waves' sums
    k = (64 + 6 + 16) * U
    sum_x = (k + 2 * U) * np.abs(x - t["mean"][:, None]).mean(1, keepdims=True)
    xh = t["rstd"][:, None] * (4 * U * np.abs(x - t["mean"][:, None]) + U * (np.abs(x) + np.abs(t["mean"])[:, None]) + sum_x)
    xh = xh + (k + 2 * (xh * np.abs(t["xhat"])).mean(1, keepdims=True) + 6 * U) * np.abs(t["xhat"])
    ady = np.abs(dy)
    eg = (ady * xh).sum(0) + (depth + 2) * U * (ady * (np.abs(t["xhat"]) + xh)).sum(0)
    eb = (depth + 2) * U * ady.sum(0)
    got = N.run(T, x, gamma, beta, dy, dtype)
    for what, off in (("dgamma", eg), ("dbeta", eb)):
        want = t[what]
        L.within(got[what], want, off + L.HALF_ULP[dtype] * (np.abs(want) + off) + L.TINY[dtype], what)
        assert np.median(off) < 0.02 * np.sqrt(np.mean(want * want))   # (nothing left out would pass)
