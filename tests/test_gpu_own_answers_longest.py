"""Drawn tokens and layer normalisation of the longest rows: a vocabulary of millions, whose whole numbers are held to fewer places, and rows of 2^24 elements."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import test_gpu_layernorm as N  # noqa: E402
import test_gpu_sample_tokens as S  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_long_vocabulary(T, dtype):
    vocab = (1 << 22) + 5
    x, u = S.logits(3, vocab, dtype, 1)
    x[1, ::2] = -np.inf
    x[2, : vocab - 3] -= 60.0
    for s in ((1.0, 0, 1.0, 0.0), (0.6, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.9, 50, 0.95, 0.01), (1.0, 100000, 1.0, 0.0)):
        S.check(T, x, u, dtype, [s] * 3, S.run(T, x, u, dtype, temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3]), f"{s}")


def test_the_longest_rows(T):
    """A row of +1 and -1 in turns and one of 3 and 5: every sum on the way is a whole number below 2^27 that fp32 holds, or one that cancels."""
    n = 1 << 24
    x = np.ones((2, n))
    x[0, 1::2] = -1
    x[1] = 3.0
    x[1, 1::2] = 5.0
    dy = np.zeros((2, n))
    dy[:, 7] = 1.0
    bx, bd, y, dx, st, dg, db = Buf(T, x), Buf(T, dy), out(T, (2, n)), out(T, (2, n)), out(T, (2, 2)), out(T, n), out(T, n)
    T.layernorm_fwd(2, n, bx, None, None, y, st, eps=N.EPS)
    r = 1 / np.sqrt(1 + np.float64(np.float32(N.EPS)))
    assert np.allclose(st.read(), [[0, r], [4, r]], rtol=4 * N.U, atol=0)
    want = np.where(np.arange(n) % 2, -r, r)
    assert np.abs(y.read() - np.stack([want, -want])).max() <= 8 * N.U
    T.layernorm_bwd(2, n, bx, None, st, bd, dx, dg, db)
    xhat = np.stack([want, -want])
    # (the two means are 2^-24 and -2^-24 or 2^-24 of a number near 1)
    g = r * (dy - 2.0 ** -24 - xhat * (xhat[:, 7] * 2.0 ** -24)[:, None])
    assert np.abs(dx.read() - g).max() <= 8 * N.U * 1.01
    assert np.abs(dx.read() - g)[:, 8:].max() <= 8 * N.U * 2.0 ** -23
    wg, wb = np.zeros(n), np.zeros(n)
    wg[7], wb[7] = (dy * xhat).sum(), 2.0
    assert np.array_equal(db.read(), wb) and np.abs(dg.read() - wg).max() <= 8 * N.U
