"""Tokens drawn from rows that are masked with their type's lowest number in the place of -inf: those logits count, behind all others, for top-k."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
import test_gpu_sample_tokens as S  # noqa: E402

pytestmark = pytest.mark.gpu

LOWEST = {"f32": float(np.finfo(np.float32).max), "bf16": float(L.decode(np.array([0x7F7F], np.uint16), "bf16")[0]), "f16": 65504.0}


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [129, 200, 500, 512, 1000, 1024, 1025, 4001, 20001, 70001])
@pytest.mark.parametrize("near", [0, 3])
def test_top_k_among_the_lowest(T, vocab, dtype, near):
    """Ten logits are left, the rest is the lowest number (near: or one of so many above it); top_k is below ten, above it and above all."""
    rng = np.random.RandomState(vocab + near)
    settings = [(t, k, p, 0.0) for k in (7, 50, min(128, vocab - 1), vocab - 1, vocab + 5) for t, p in ((1.0, 1.0), (0.9, 0.9), (np.inf, 1.0), (np.inf, 0.8))]
    rows = len(settings)
    low = L.encode(np.full((rows, vocab), -LOWEST[dtype]), dtype)
    if near:
        low = low - rng.randint(0, near + 1, low.shape).astype(low.dtype) if dtype != "f32" else (
            low.view(np.uint32) - rng.randint(0, near + 1, low.shape).astype(np.uint32)).view(np.float32)
    x = L.decode(low, dtype)
    for r in range(rows):
        at = rng.choice(vocab, 10, replace=False)
        x[r, at] = L.rounded(2 * rng.randn(10), dtype)
    u = np.float32(rng.rand(rows))
    S.check(T, x, u, dtype, settings, S.run(T, x, u, dtype, settings), f"{vocab} {dtype}")
