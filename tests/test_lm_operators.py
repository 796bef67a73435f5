"""The language-model operators without a GPU: what they refuse, before anything reaches a device, and the tests' own
64-bit forms against published values and differences."""
import ctypes as C
import importlib
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402


@pytest.fixture(scope="module")
def T():
    return importlib.import_module("tiny-cnn_amd")


class At:
    """An address that no call may follow."""

    def __init__(self, address):
        self.ptr = C.c_void_p(address)


A, B, D = At(0x100000000), At(0x200000000), At(0x300000000)


def refuses(T, what, f, *args, **kw):
    with pytest.raises(T.TdhError, match=r"\[-1\].*" + what):
        f(*args, **kw)


def test_gated_ff_refusals(T):
    ok = dict(act="silu", dtype="f32")
    refuses(T, "bad shape", T.gated_ff_fwd, 0, 8, False, 1, A, B, None, D, **ok)
    refuses(T, "bad shape", T.gated_ff_fwd, 8, -1, False, 1, A, B, None, D, **ok)
    refuses(T, "bad shape", T.gated_ff_fwd, 8, 8, False, -1, A, B, None, D, **ok)
    refuses(T, "null tensor", T.gated_ff_fwd, 8, 8, False, 1, None, B, None, D, **ok)
    refuses(T, "has_bias", T.gated_ff_fwd, 8, 8, True, 1, A, B, None, D, **ok)
    refuses(T, "2\\^31", T.gated_ff_fwd, 1 << 16, 1 << 15, False, 1, A, B, None, D, **ok)
    for shape in ((1 << 22, 1, 1), (1, 1 << 21, 1), (1, 1, 1 << 25), (1, 1, (1 << 20) + 1)):
        refuses(T, "beyond", T.gated_ff_fwd, shape[0], shape[1], False, shape[2], A, B, None, D, **ok)
        refuses(T, "beyond", T.gated_ff_bwd, shape[0], shape[1], False, shape[2], A, B, D, D, None, D, None, **ok)
    far, near = At(0x500000000), At(0x500000000 + 4 * 64)
    refuses(T, "overlaps an input", T.gated_ff_fwd, 8, 16, False, 8, A, far, None, near, **ok)
    refuses(T, "two outputs overlap", T.gated_ff_fwd, 8, 16, False, 8, A, B, None, far, z=near, **ok)
    refuses(T, "overlaps an input", T.gated_ff_bwd, 8, 16, False, 8, A, B, D, far, near, None, None, **ok)
    refuses(T, "two outputs overlap", T.gated_ff_bwd, 8, 16, False, 8, A, B, D, At(0x700000000), near, far, None, **ok)
    refuses(T, "aligned", T.gated_ff_fwd, 8, 8, False, 1, At(0x100000001), B, None, D, act="silu", dtype="bf16")
    refuses(T, "aligned", T.gated_ff_fwd, 8, 8, False, 1, A, B, None, D, z=At(0x300000002), act="silu", dtype="bf16")
    refuses(T, "null tensor", T.gated_ff_bwd, 8, 8, False, 1, A, B, None, D, None, None, None, **ok)
    lib = T.lib()
    assert lib.tdh_gated_ff_fwd(3, 0, 8, 8, 0, 1, A.ptr, B.ptr, None, D.ptr, None) == -1
    assert b"element type" in lib.tdh_last_error()
    assert lib.tdh_gated_ff_fwd(0, 6, 8, 8, 0, 1, A.ptr, B.ptr, None, D.ptr, None) == -1
    assert b"activation" in lib.tdh_last_error()


def test_dropout_refusals(T):
    for rate in (-0.1, 1.0, 1.5, float("nan")):
        refuses(T, "rate", T.dropout_seeded_fwd, 8, A, B, rate, 1)
        refuses(T, "rate", T.dropout_seeded_bwd, 8, A, B, rate, 1)
    refuses(T, "null tensor", T.dropout_seeded_fwd, 8, None, B, 0.5, 1)
    refuses(T, "null tensor", T.dropout_seeded_bwd, 8, A, None, 0.5, 1)
    refuses(T, "aligned", T.dropout_seeded_fwd, 8, A, At(0x200000002), 0.5, 1)
    refuses(T, "aligned", T.dropout_seeded_fwd, 8, A, B, 0.5, 1, residual=At(0x300000001), dtype="f16")
    refuses(T, "overlaps", T.dropout_seeded_fwd, 8, A, At(0x100000004), 0.5, 1)
    refuses(T, "overlaps", T.dropout_seeded_fwd, 8, A, B, 0.5, 1, residual=At(0x200000010))
    refuses(T, "elements", T.dropout_seeded_fwd, (1 << 62), A, B, 0.5, 1)


def test_loss_refusals(T):
    one = dict(rows=4, vocab=8, logits=A, target=B)
    refuses(T, "rows of", T.token_logprob_fwd, -1, 8, A, B, D)
    refuses(T, "rows of", T.token_logprob_fwd, 4, 0, A, B, D)
    refuses(T, "elements apart", T.token_logprob_fwd, 4, 8, A, B, D, ld=7)
    refuses(T, "null tensor", T.token_logprob_fwd, 4, 8, None, B, D)
    refuses(T, "null tensor", T.token_logprob_fwd, 4, 8, A, B, None)
    refuses(T, "aligned", T.token_logprob_fwd, 4, 8, At(0x100000001), B, D, dtype="bf16")
    refuses(T, "null tensor", T.token_logprob_bwd, 4, 8, A, B, None, D, At(0x400000000))
    refuses(T, "elements apart", T.token_logprob_bwd, 4, 8, A, B, D, D, At(0x400000000), ld_d=7)
    refuses(T, "overlaps", T.token_logprob_bwd, 4, 8, A, B, D, D, At(0x100000020))
    refuses(T, "overlaps", T.token_logprob_bwd, 4, 8, A, B, D, D, A, ld_d=16)
    refuses(T, "clipping", T.policy_loss, old_logp=D, ref_logp=None, advantage=D, clip_low=-0.1, **one)
    refuses(T, "clipping", T.policy_loss, old_logp=D, ref_logp=None, advantage=D, clip_low=1.5, **one)
    refuses(T, "clipping", T.policy_loss, old_logp=D, ref_logp=None, advantage=D, clip_high=float("inf"), **one)
    refuses(T, "KL", T.policy_loss, old_logp=D, ref_logp=None, advantage=D, kl_coef=float("nan"), **one)
    refuses(T, "null tensor", T.policy_loss, old_logp=None, ref_logp=None, advantage=D, **one)
    refuses(T, "beta", T.preference_loss, 1, seq_start=D, beta=0.0, **one)
    refuses(T, "smoothing", T.preference_loss, 1, seq_start=D, smoothing=1.5, **one)
    refuses(T, "pairs", T.preference_loss, -1, seq_start=D, **one)
    refuses(T, "null tensor", T.preference_loss, 1, seq_start=None, **one)
    p = T.PreferenceDesc(3, 0.1, 0.0)
    assert T.lib().tdh_preference_loss(C.byref(p), 0, 1, 4, 8, A.ptr, C.c_size_t(8), B.ptr, D.ptr, None, None, None, None, None,
                                       None, C.c_size_t(8)) == -1
    assert b"kind" in T.lib().tdh_last_error()
    assert T.lib().tdh_policy_loss(None, 0, 4, 8, A.ptr, C.c_size_t(8), B.ptr, D.ptr, None, D.ptr, None, None, None, None, None,
                                   C.c_size_t(8)) == -1


def test_loss_refusals_of_overlapping_tensors(T):
    one = dict(rows=4, vocab=8, logits=A, target=B)
    refuses(T, "overlaps an input", T.token_logprob_fwd, 4, 8, A, B, At(B.ptr.value + 12))
    refuses(T, "two outputs overlap", T.token_logprob_fwd, 4, 8, A, B, D, stats=At(D.ptr.value + 12))
    refuses(T, "overlaps an input", T.token_logprob_bwd, 4, 8, A, B, D, At(0x400000000), At(D.ptr.value + 28))
    refuses(T, "overlaps an input", T.policy_loss, old_logp=D, ref_logp=None, advantage=At(0x400000000), logp=D, **one)
    refuses(T, "overlaps an input", T.policy_loss, old_logp=D, ref_logp=None, advantage=D, loss=At(A.ptr.value + 124), **one)
    refuses(T, "overlaps an input", T.preference_loss, 1, seq_start=D, ref_logp=At(0x400000000), seq_logp=At(0x400000004), **one)
    refuses(T, "two outputs overlap", T.preference_loss, 1, seq_start=D, margin=At(0x400000000), loss=At(0x400000000), **one)


def test_cast_refusals(T):
    refuses(T, "null tensor", T.cast, 4, None, B, "f32", "bf16")
    refuses(T, "overlap", T.cast, 4, A, At(0x100000008), "f32", "bf16")
    refuses(T, "overlap", T.cast, 4, A, A, "bf16", "f32")
    refuses(T, "aligned", T.cast, 4, At(0x100000002), B, "f32", "bf16")


def test_descriptors_match_the_header(T, tmp_path):
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "s.c").write_text('#include <stdio.h>\n#include "tdh.h"\nint main(void) { printf("%zu %zu", '
                                  'sizeof(tdh_policy_desc), sizeof(tdh_preference_desc)); return 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), "-o", str(tmp_path / "s"), str(tmp_path / "s.c")],
                   check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == [C.sizeof(T.PolicyDesc), C.sizeof(T.PreferenceDesc)]


def test_generator_against_published_values():
    """The known answers that the generator's authors publish with it (counter, key -> four words)."""
    assert [hex(v) for v in L.philox_words(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def test_mask_share():
    """A share `rate` is dropped: 10^6 draws, five standard deviations."""
    for rate in (0.1, 0.5, 0.9):
        dropped = 1.0 - L.kept(10 ** 6, rate, 1234567890123456789, 77).mean()
        assert abs(dropped - rate) < 5 * np.sqrt(rate * (1 - rate) / 1e6)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "sigmoid", "relu", "none"])
def test_gated_ff_gradient_by_differences(act):
    rng = np.random.RandomState(1)
    x, w, b, dh = rng.randn(3, 5), rng.randn(5, 8), rng.randn(8), rng.randn(3, 4)
    z, _ = L.ff_forward(x, w, b, act)
    _, dx, dw, db = L.ff_backward(x, w, z, dh, act)
    eps = 1e-6
    for name, v, grad in (("x", x, dx), ("w", w, dw), ("b", b, db)):
        for i in np.ndindex(v.shape):
            keep = v[i]
            v[i] = keep + eps
            up = (L.ff_forward(x, w, b, act)[1] * dh).sum()
            v[i] = keep - eps
            down = (L.ff_forward(x, w, b, act)[1] * dh).sum()
            v[i] = keep
            assert abs((up - down) / (2 * eps) - grad[i]) < 1e-6 * (1 + abs(grad[i])), (name, i)


def test_policy_gradient_by_differences():
    rng = np.random.RandomState(2)
    x, target = rng.randn(6, 9), np.array([0, 8, -1, 3, 4, 5])
    now = L.logprob(x, target)[0]
    old, ref, adv, w = now + 0.1 * rng.randn(6), now + 0.3 * rng.randn(6), rng.randn(6), rng.rand(6)

    def loss(x):
        return L.policy(L.logprob(x, target)[0], target, old, ref, adv, w, 0.2, 0.3, 0.1)[0].sum()

    d = L.policy(now, target, old, ref, adv, w, 0.2, 0.3, 0.1)[1]
    grad = L.dlogits(x, target, d)
    by_differences(loss, x, grad)


def by_differences(loss, x, grad, eps=1e-6):
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + eps
        up = loss(x)
        x[i] = keep - eps
        down = loss(x)
        x[i] = keep
        assert abs((up - down) / (2 * eps) - grad[i]) < 1e-7 + 1e-6 * abs(grad[i]), i


@pytest.mark.parametrize("kind", ["sigmoid", "squared", "hinge"])
def test_preference_gradient_by_differences(kind):
    rng = np.random.RandomState(3)
    start, target = np.array([0, 3, 4, 6, 9]), np.array([1, -1, 2, 0, 4, 4, 3, 2, 1])
    x, ref = rng.randn(9, 5), rng.randn(4)
    seq = np.repeat(np.arange(4), np.diff(start))

    def total(x):
        return np.bincount(seq, L.logprob(x, target)[0], minlength=4)

    d = L.preference(total(x), ref, 0.4, 0.1, kind)[2]
    by_differences(lambda v: L.preference(total(v), ref, 0.4, 0.1, kind)[1].mean(), x, L.dlogits(x, target, d[seq]))
