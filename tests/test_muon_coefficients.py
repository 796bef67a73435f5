"""Which coefficients the orthogonalised update refuses: those that take a singular value of at most 1 beyond 4 in any step. Matrices without elements, so that
nothing reaches a device."""
import ctypes as C
import importlib

import numpy as np
import pytest


@pytest.fixture(scope="module")
def T():
    return importlib.import_module("tiny-cnn_amd")


def accepted(T, a, b, c, steps):
    o = T.muon_desc(a=a, b=b, c=c, steps=steps)
    rc = T.lib().tdh_orthogonalize(C.byref(o), 0, 0, 0, None, None)
    return not (rc != 0 and b"coefficients" in T.lib().tdh_last_error())


def largest(a, b, c, steps):
    """The largest singular value after each step, by 20001 samples of its range: of a polynomial of degree 5 they miss a maximum by a part in 10^6."""
    a, b, c = (float(np.float32(v)) for v in (a, b, c))
    most, out = 1.0, []
    for _ in range(steps):
        s = most * np.linspace(0, 1, 20001)
        most = np.abs(s * (a + b * s ** 2 + c * s ** 4)).max()
        out.append(most)
        if most > 100:
            break
    return out


# the last term is so small beside the others that the turning points' formula has to keep its figures
@pytest.mark.parametrize("c", [0.0, 1e-20, -1e-20, 1e-38, -1e-38, 1e-12, -1e-9, 1e-5])
def test_a_small_last_coefficient(T, c):
    assert accepted(T, 10.0, -10.0, c, 1)         # 10 (s - s^3) is 3.85 at s^2 = 1/3 ...
    assert not accepted(T, 10.0, -10.0, c, 2)     # ... and -531 of that
    assert accepted(T, 1.5, -0.5, c, 32)          # the cubic that converges to one
    assert accepted(T, -10.0, 10.0, c, 1) and not accepted(T, -10.0, 10.0, c, 2)


def test_against_samples(T):
    rng = np.random.RandomState(5)
    borders = 0
    for i in range(600):
        a, b, c = rng.randn(3) * np.array([4, 8, 8]) * rng.choice([1e-6, 0.1, 0.5, 1, 1], 3)
        if i % 7 == 0:
            c = rng.choice([0.0, 1e-30, -1e-25, 1e-15])
        if i % 11 == 0:
            b = 0.0
        steps = int(rng.choice([1, 2, 5]))
        most = max(largest(a, b, c, steps))
        if abs(most - 4) < 1e-3:
            borders += 1
            continue
        assert accepted(T, a, b, c, steps) == (most < 4), (a, b, c, steps, most)
    assert borders < 20
    assert accepted(T, 3.4445, -4.7750, 2.0315, 32)
    assert accepted(T, 0.0, 0.0, 0.0, 3) and accepted(T, 4.0, 0.0, 0.0, 1) and not accepted(T, 4.001, 0.0, 0.0, 1)
