"""Tokens drawn without filters from long rows at temperatures of a logit's last place."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import test_gpu_sample_tokens as S  # noqa: E402

pytestmark = pytest.mark.gpu

US = np.array([0.0, 1e-5, 0.0003, 0.001, 0.0015, 0.01, 0.3, 0.5, 0.9, 0.999], np.float32)


# (logit, temperature): 4 temperatures are a half to one and a half of the logit's last place, and the next number's weight is e^5 to e^8
@pytest.mark.parametrize("at,temperature", [(100.0, 1e-6), (6000.0, 7e-5), (70000.0, 1.1e-3), (6e5, 0.01), (-100.0, 1e-6), (1e30, 1.2e22), (2.0 ** 100, 3e22)])
@pytest.mark.parametrize("rows", [1, 60])
def test_a_last_place_apart(T, at, temperature, rows):
    """The maximum lies one place above the largest of what a row's threads look at first: a thread's words are 64 apart, so word 1030 is nobody's
    first with 512 threads or 1024."""
    vocab, n = 9001, 10 * rows
    rng = np.random.RandomState(3)
    x = np.full((n, vocab), -np.inf)
    low = np.float32(at)
    up = np.nextafter(low, np.float32(np.inf))
    x[:, 0] = low
    x[:, 4 * 1030 + 1] = up
    for v in (low, np.nextafter(low, np.float32(-np.inf))):   # (every other row: more of the lower ones behind it, and some below)
        x[1::2, rng.randint(4200, vocab, 300)] = v
    u = np.repeat(US, rows)
    got = S.run(T, x, u, "f32", temperature=temperature)
    some = np.arange(0, n, max(1, rows // 2 - 1))
    S.check(T, x[some], u[some], "f32", [(temperature, 0, 1.0, 0.0)] * len(some), [g[some] for g in got], f"{at} {temperature}")


@pytest.mark.parametrize("temperature", [1e-7, 1e-6, 3e-6, 1e-5, 1e-4, 1e-3])
@pytest.mark.parametrize("at", [3.0, 40.0, 500.0, 9000.0])
def test_steps_of_a_last_place(T, at, temperature):
    """Logits up to twelve places around one number."""
    rng = np.random.RandomState(int(at))
    ulp = float(np.spacing(np.float32(at)))
    x = np.float32(at + ulp * rng.randint(-12, 13, (40, 5003))).astype(np.float64)
    x[:, ::2] = at - 12 * ulp
    x[20:, 4 * 64:] += 3 * ulp
    u = np.float32(rng.rand(40))
    S.check(T, x, u, "f32", [(temperature, 0, 1.0, 0.0)] * 40, S.run(T, x, u, "f32", temperature=temperature), f"{at} {temperature}")
