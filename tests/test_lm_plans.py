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


class At:
    """An address that no call may follow."""

    def __init__(self, address):
        self.ptr = C.c_void_p(address)


@pytest.mark.parametrize("dtype,longest", [("f32", 16376), ("bf16", 32752), ("f16", 32752)])
def test_long_rows_are_as_many_as_a_launch_has_threads_for(dtype, longest):
    """A row of more than 4096 words gets up to 1024 threads, and 2^22 such rows are 2^32 threads, where a launch's number wraps and
    it does nothing of the work without an error. (Calls that are not refused for that end where the library is not initialised, or at
    a null tensor.)"""
    a, b, d = At(1 << 44), At(1 << 45), At(1 << 46)
    calls = {"logprob": lambda rows, v, t: T.token_logprob_fwd(rows, v, a, b, t, dtype=dtype),
             "logprob_bwd": lambda rows, v, t: T.token_logprob_bwd(rows, v, a, b, d, d, t, dtype=dtype),
             "policy": lambda rows, v, t: T.policy_loss(rows, v, a, b, t, None, d, dtype=dtype),
             "preference": lambda rows, v, t: T.preference_loss(1, rows, v, a, b, t, dtype=dtype)}
    for call in calls.values():
        with pytest.raises(T.TdhError, match="64 KB"):
            call(1 << 22, longest + 1, None)
        for rows, v in (((1 << 22) - 1, longest + 1), (1 << 22, longest)):
            with pytest.raises(T.TdhError, match="null tensor|too many"):
                call(rows, v, None)


def test_no_kernel_of_the_losses_that_nothing_launches():
    """The row kernels that the library holds, by how many waves and words they have: log-probabilities of rows past 4096 words
    are read as they come, and the policy loss never reads past the caches."""
    import re
    with open(os.path.join(os.path.dirname(T.__file__), "lib", "libtdh.so"), "rb") as f:
        names = set(re.findall(rb"row_kernelI[A-Za-z0-9_]+?Li(\d)ELi(\d+)ELi(\d+)ELb([01])EEEvNS", f.read()))
    got = {tuple(int(v) for v in n) for n in names}
    both = {(1, 1), (1, 2), (1, 4), (1, 8), (4, 4), (4, 8), (4, 16), (16, 0), (16, 1), (16, 4)}
    assert got == {(m, w, k, 0) for m in (0, 1) for w, k in both} | {(0, 8, 0, 0), (0, 8, 0, 1), (1, 16, 8, 0), (1, 16, 16, 0)}


def test_assembly_that_writes_m0_leaves_it_as_it_was():
    """The compiler keeps m0 for itself (named as clobbered it is warned about and no more)."""
    import glob
    import re
    found = 0
    for path in glob.glob(os.path.join(os.path.dirname(T.__file__), "csrc", "*.h*")):
        with open(path) as f:
            for asm in re.findall(r"asm\s+volatile\s*\((.*?)\);", f.read(), re.S):
                if "s_mov_b32 m0" in asm:
                    found += 1
                    text = "".join(re.findall(r'"([^"]*)"', asm.split("\n")[0])).replace("\\n\\t", "\n").split("\n")
                    assert text[0] == "s_mov_b32 %0, m0" and text[-1] == "s_mov_b32 m0, %0" and '"=&s"' in asm, (path, asm)
    assert found


class FfPlan(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("cfg", "splits", "k_per_split")]


def test_the_gpu_tests_reach_every_tile_of_the_16_bit_products():
    """Forward, input and weight gradient, each on all five tiles, split along the reduction and whole."""
    import test_gpu_lm_sizes as sizes
    f = T.lib()._ZN3tdh7ff_planEiiib   # tdh::ff_plan
    f.restype, f.argtypes = FfPlan, [C.c_int] * 3 + [C.c_bool]
    for aligned in (False, True):
        reached = set()
        for n, d, h in sizes.TILE_SHAPES:
            half = (h + 7) & ~7
            d = (d + 7) & ~7 if aligned else d
            for product, plan in (("forward", f(n, 2 * half, d, True)), ("dx", f(n, d, 2 * half, False)), ("dw", f(d, 2 * half, n, False))):
                reached.add((product, plan.cfg, plan.splits > 1))
        missing = {(p, c, s) for p in ("forward", "dx", "dw") for c in range(5) for s in (False, True)} - reached
        assert not missing, (aligned, missing)
