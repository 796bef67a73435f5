"""Which kernels the operators of language models come to (host code, no GPU): limits of a launch, and that the GPU tests reach every tile."""
import ctypes as C
import importlib
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

T = importlib.import_module("tiny-cnn_amd")


class GemmPlan(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("cfg", "bm", "bn", "splits", "k_per_split")]


def plan_gemm(m, n, k, split):
    f = T.lib()._ZN3tdh9plan_gemmEiiib   # tdh::plan_gemm
    f.restype, f.argtypes = GemmPlan, [C.c_int, C.c_int, C.c_int, C.c_bool]
    return f(m, n, k, split)


@pytest.mark.parametrize("split", [False, True])
def test_fully_connected_products_have_no_more_tiles_of_rows_than_a_launch_takes(split):
    """A launch takes 65535 workgroups along y, where a product has its tiles of rows: the weight gradient of up to 2^21 inputs."""
    for m in (1 << 20, 65535 * 32, 65535 * 32 + 1, (1 << 21) - 1, 1 << 21, 1 << 22):
        for n in (1, 2, 4, 8, 16, 32, 40, 64, 128, 256, 500):
            for k in range(1, 40):
                p = plan_gemm(m, n, k, split)
                assert -(-m // p.bm) <= 65535, (m, n, k, p.cfg)
