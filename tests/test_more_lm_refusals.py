"""What layer normalisation, the orthogonalised update, token sampling and products in 8-bit integers refuse, before anything reaches a
device."""
import ctypes as C
import importlib
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_lm_operators import A, B, D, At, refuses  # noqa: E402


@pytest.fixture(scope="module")
def T():
    return importlib.import_module("tiny-cnn_amd")


F, G = At(0x400000000), At(0x500000000)


def test_layernorm_refusals(T):
    fwd, bwd = T.layernorm_fwd, T.layernorm_bwd
    refuses(T, "rows of", fwd, -1, 8, A, B, B, D)
    refuses(T, "rows of", fwd, 4, 0, A, B, B, D)
    refuses(T, "rows of", fwd, 1 << 24, 8, A, B, B, D)
    refuses(T, "rows of", bwd, 4, (1 << 24) + 1, A, None, F, D, G, None, None)
    for eps in (0.0, -1e-5, 1e-42, float("inf"), float("nan")):
        refuses(T, "eps", fwd, 4, 8, A, B, B, D, eps=eps)
    refuses(T, "null tensor", fwd, 4, 8, None, B, B, D)
    refuses(T, "null tensor", fwd, 4, 8, A, B, B, None)
    refuses(T, "null tensor", bwd, 4, 8, A, None, None, D, G, None, None)
    refuses(T, "null tensor", bwd, 4, 8, A, None, F, None, G, None, None)
    refuses(T, "of x 7 apart", fwd, 4, 8, A, B, B, D, ld=7)
    refuses(T, "of y 7 apart", fwd, 4, 8, A, B, B, D, ld_y=7)
    refuses(T, "of dy 7 apart", bwd, 4, 8, A, None, F, D, G, None, None, ld_dy=7)
    refuses(T, "of dx 7 apart", bwd, 4, 8, A, None, F, D, G, None, None, ld_dx=7)
    refuses(T, "aligned", fwd, 4, 8, At(A.ptr.value + 1), B, B, D, dtype="f16")
    refuses(T, "aligned", fwd, 4, 8, A, At(B.ptr.value + 1), B, D, dtype="f16")
    refuses(T, "aligned", fwd, 4, 8, A, B, B, D, At(F.ptr.value + 2), dtype="f16")
    refuses(T, "aligned", bwd, 4, 8, A, None, F, D, G, At(B.ptr.value + 2), None)
    refuses(T, "overlaps an input", fwd, 4, 8, A, B, B, At(A.ptr.value + 4))
    refuses(T, "overlaps an input", fwd, 4, 8, A, B, B, A, ld=16)
    refuses(T, "overlaps an input", fwd, 4, 8, A, B, B, B)
    refuses(T, "overlaps an input", fwd, 4, 8, A, B, B, D, At(A.ptr.value + 120))
    refuses(T, "two outputs overlap", fwd, 4, 8, A, B, B, D, At(D.ptr.value + 120))
    refuses(T, "overlaps an input", bwd, 4, 8, A, None, F, D, A, None, None)
    refuses(T, "overlaps an input", bwd, 4, 8, A, None, F, D, At(D.ptr.value + 4), None, None)
    refuses(T, "overlaps an input", bwd, 4, 8, A, None, F, D, G, At(D.ptr.value + 8), None)
    refuses(T, "two outputs overlap", bwd, 4, 8, A, None, F, D, None, G, At(G.ptr.value + 28))
    assert T.lib().tdh_layernorm_fwd(3, 4, 8, C.c_float(1e-5), A.ptr, C.c_size_t(8), None, None, D.ptr, C.c_size_t(8), None) == -1
    assert b"element type" in T.lib().tdh_last_error()


def test_sample_refusals(T):
    f, one = T.sample_tokens, (4, 8, A, B, D)
    refuses(T, "rows of", f, -1, 8, A, B, D)
    refuses(T, "rows of", f, 1 << 22, 8, A, B, D)
    refuses(T, "rows of", f, 4, 0, A, B, D)
    refuses(T, "rows of", f, 4, (1 << 30) + 1, A, B, D)
    refuses(T, "elements apart", f, *one, ld=7)
    for i in (2, 3, 4):
        refuses(T, "null tensor", f, *[None if i == k else v for k, v in enumerate(one)])
    for t in (-0.5, float("inf"), float("nan")):
        refuses(T, "temperature", f, *one, temperature=t)
    refuses(T, "top_k", f, *one, top_k=-1)
    for p in (0.0, 1.5, float("nan")):
        refuses(T, "top_p", f, *one, top_p=p)
    for q in (-0.1, 1.5, float("nan")):
        refuses(T, "min_p", f, *one, min_p=q)
    refuses(T, "aligned", f, 4, 8, At(A.ptr.value + 1), B, D, dtype="bf16")
    refuses(T, "aligned", f, 4, 8, A, B, D, logp=At(F.ptr.value + 2), dtype="bf16")
    refuses(T, "overlaps an input", f, 4, 8, A, B, At(A.ptr.value + 124))
    refuses(T, "overlaps an input", f, 4, 8, A, B, D, logq=B)
    refuses(T, "overlaps an input", f, 4, 8, A, B, D, settings=F, kept=At(F.ptr.value + 60))
    refuses(T, "two outputs overlap", f, 4, 8, A, B, D, logp=At(D.ptr.value + 12))
    assert T.lib().tdh_sample_tokens(None, None, 0, 4, 8, A.ptr, C.c_size_t(8), B.ptr, D.ptr, None, None, None) == -1
    assert b"descriptor" in T.lib().tdh_last_error()


def test_muon_refusals(T):
    d = T.muon_desc
    refuses(T, "bad shape", T.orthogonalize, d(), -1, 8, A, B)
    refuses(T, "beyond", T.orthogonalize, d(), 16385, 16385, A, B)
    refuses(T, "beyond", T.orthogonalize, d(), 1, (1 << 20) + 1, A, B)
    refuses(T, "beyond", T.orthogonalize, d(), 1 << 20, 1025, A, B)
    refuses(T, "null tensor", T.orthogonalize, d(), 8, 8, None, B)
    refuses(T, "null tensor", T.orthogonalize, d(), 8, 8, A, None)
    refuses(T, "null tensor", T.muon_update, d(), 8, 8, A, B, None)
    refuses(T, "aligned", T.orthogonalize, d(), 8, 8, At(A.ptr.value + 1), B, dtype="f16")
    refuses(T, "aligned", T.muon_update, d(), 8, 8, A, At(B.ptr.value + 2), D, dtype="f16")
    refuses(T, "overlaps an input", T.orthogonalize, d(), 8, 8, A, At(A.ptr.value + 4))
    refuses(T, "overlaps an input", T.muon_update, d(), 8, 8, A, B, At(A.ptr.value + 252))
    refuses(T, "two outputs overlap", T.muon_update, d(), 8, 8, A, B, At(B.ptr.value + 252))
    refuses(T, "steps", T.orthogonalize, d(steps=33), 8, 8, A, B)
    refuses(T, "steps", T.orthogonalize, d(steps=-1), 8, 8, A, B)
    for eps in (0.0, float("nan"), float("inf"), 1e-42):
        refuses(T, "eps", T.orthogonalize, d(eps=eps), 8, 8, A, B)
    for k in (dict(a=5.0), dict(b=1.0), dict(c=float("nan")), dict(a=float("inf")), dict(a=3.0, b=0.5, c=0.0)):
        refuses(T, "coefficients", T.orthogonalize, d(**k), 8, 8, A, B)
    refuses(T, "products", T.orthogonalize, d(products="bf16"), 8, 8, A, B)
    assert T.lib().tdh_orthogonalize(None, 0, 8, 8, A.ptr, B.ptr) == -1
    o = d()
    assert T.lib().tdh_muon_update(C.byref(o), 3, 8, 8, A.ptr, C.c_float(1.0), B.ptr, D.ptr) == -1
    assert b"element type" in T.lib().tdh_last_error()


def test_q8_refusals(T):
    f, one = T.fc_q8_fwd, (64, 8, False, 4, A, B, F, None, D)
    refuses(T, "bad shape", f, 0, *one[1:])
    refuses(T, "bad shape", f, 64, 0, *one[2:])
    refuses(T, "beyond", f, (1 << 17) + 1, *one[1:])
    refuses(T, "beyond", f, 64, (1 << 20) + 1, *one[2:])
    refuses(T, "samples", f, 64, 8, False, -1, *one[4:])
    refuses(T, "samples", f, 64, 8, False, (1 << 24) + 1, *one[4:])
    refuses(T, "2\\^31", f, 1 << 17, 1 << 14, *one[2:])
    refuses(T, "2\\^31", f, 64, 1 << 10, False, 1 << 21, *one[4:])
    for i in (4, 5, 6, 8):
        refuses(T, "null tensor", f, *[None if i == k else v for k, v in enumerate(one)])
    refuses(T, "has_bias", f, 64, 8, True, *one[3:])
    refuses(T, "16-byte", f, 64, 8, False, 4, A, At(B.ptr.value + 8), F, None, D)
    refuses(T, "aligned", f, 64, 8, False, 4, At(A.ptr.value + 1), B, F, None, D, dtype="bf16")
    refuses(T, "aligned", f, 64, 8, False, 4, A, B, At(F.ptr.value + 2), None, D, dtype="bf16")
    refuses(T, "overlaps an input", f, 64, 8, False, 4, A, B, F, None, At(A.ptr.value + 1020))
    refuses(T, "overlaps an input", f, 64, 8, False, 4, A, B, F, None, At(B.ptr.value + 508))
    p = T.fc_q8_pack
    refuses(T, "bad shape", p, -3, 8, A, B, D)
    refuses(T, "null tensor", p, 64, 8, A, None, D)
    refuses(T, "16-byte", p, 64, 8, A, At(B.ptr.value + 4), D)
    refuses(T, "overlaps an input", p, 64, 8, A, At(A.ptr.value + 64), D)
    refuses(T, "two outputs overlap", p, 64, 8, A, B, At(B.ptr.value + 500))
    assert T.q8_row(0) == 0 and T.q8_row(1) == 16 and T.q8_row(16) == 16 and T.q8_row(17) == 32
    assert T.lib().tdh_fc_q8_fwd(7, 64, 8, 0, 4, A.ptr, B.ptr, F.ptr, None, D.ptr) == -1
    assert b"element type" in T.lib().tdh_last_error()
