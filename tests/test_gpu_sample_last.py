"""A random number of 1 or more counts as the largest fp32 number below 1, 1 - 2^-24: a token with less than that of all is not drawn behind the others."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import test_gpu_sample_tokens as S  # noqa: E402

pytestmark = pytest.mark.gpu

BELOW = np.nextafter(np.float32(1), np.float32(0))


@pytest.mark.parametrize("vocab", [12, 500, 3000, 9001, 70001])
@pytest.mark.parametrize("s", [(1.0, 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (1.0, 0, 0.9999999, 0.0), (1.0, 0, 1.0, 1e-30)])
def test_one_and_more(T, vocab, s):
    u = np.array([1.0, 2.0, np.inf, BELOW], np.float32)
    x = np.full((4, vocab), -np.inf)
    x[:, 1], x[:, 4], x[:, vocab - 3] = 0.0, -1.0, -20.0    # (2e-9 of them all)
    for got in (S.run(T, x, u, "f32", [s] * 4), S.run(T, x, u, "f32", temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3])):
        S.check(T, x, np.full(4, BELOW), "f32", [s] * 4, got)
        assert (got[0] == 4).all()
