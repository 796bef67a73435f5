"""Several steps of the orthogonalised update against 64 bits: no further off than the roundings that the interface names, made in numpy, take the same chain."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402
from test_gpu_muon import a, b, c, start, step  # noqa: E402

pytestmark = pytest.mark.gpu


def matrix(rows, cols, kind):
    rng = np.random.RandomState(rows + 3 * cols)
    u = rng.randn(rows, cols)
    if kind == "falling":      # some strong directions of falling strength, as gradients have
        u = 3 * (rng.randn(rows, 16) * np.logspace(0, -2, 16)) @ rng.randn(16, cols) + 0.3 * u
    elif kind == "few":        # four directions and little beside them, which grows 3.4-fold a step, and what is off beside the four with it
        u = rng.randn(rows, 4) @ rng.randn(4, cols) + 1e-3 * u
    elif kind == "flat":       # all singular values equal
        q = np.linalg.qr(rng.randn(max(rows, cols), min(rows, cols)))[0]
        u = q if rows > cols else q.T
    return L.rounded(1e-3 * u, "f32")


def f16_step(x, flat):
    """A step (no more rows than columns) with the operands of its three products rounded to fp16, X itself to two such parts."""
    half = lambda v, scale: (v * scale).astype(np.float16).astype(np.float64) / scale  # noqa: E731
    hi = half(x, 2.0 ** 14)
    g = half(hi @ hi.T - flat * np.eye(len(x)), 2.0 ** 13)
    p = half((b + 2 * c * flat) * g + c * g @ g, 2.0 ** 12)
    return (a + b * flat + c * flat * flat) * (hi + half(x - hi, 2.0 ** 14)) + p @ hi


def f32_step(x):
    a32, b32, c32 = (np.float32(v) for v in (a, b, c))
    g = x @ x.T
    return a32 * x + (b32 * g + c32 * (g @ g)) @ x


@pytest.mark.parametrize("shape", [(600, 400), (300, 129), (257, 640), (130, 1500), (1000, 130), (120, 84)])
@pytest.mark.parametrize("kind", ["gauss", "falling", "few", "flat"])
def test_steps(T, shape, kind):
    """TDH_F16: what numpy's chain is off by comes from as many roundings of the same sizes, but not the same ones where a sum's last bits differ: half as much again.
    TDH_F32: products as precise as those in fp32, whose sums are added up in some other order: twice. Beside either what sums, the start and the result round."""
    u = matrix(*shape, kind)
    x = start(u)
    x = x if shape[0] <= shape[1] else x.T
    rough16, rough32 = x, np.float32(x)
    flat, y = 1.0 / min(shape), out(T, shape)
    for k in range(6):
        rough16, rough32, x = f16_step(rough16, flat), f32_step(rough32), step(x)
        r = np.sqrt(flat)
        flat = (r * (a + b * flat + c * flat * flat)) ** 2
        if k + 1 not in (2, 5, 6):
            continue
        size = np.linalg.norm(x)
        for products, rough, more, rest in (("f16", rough16, 1.5, 2.0 ** -17), ("f32", rough32, 2.0, 2.0 ** -20)):
            T.orthogonalize(T.muon_desc(steps=k + 1, products=products), *shape, Buf(T, u), y)
            got = np.linalg.norm(y.read() - (x if shape[0] <= shape[1] else x.T)) / size
            may = np.linalg.norm(rough - x) / size
            assert got <= more * may + rest
