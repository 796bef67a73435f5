"""The language-model operators at the sizes where another kernel takes over, and at their limits, against the definitions in 64 bits."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


def whole_numbers(rng, shape, most):
    """Whole numbers, so few that sums of their products are exact in fp32: one term lost or taken twice shows."""
    return rng.randint(-most, most + 1, shape).astype(np.float64)


def ff_exact_case(T, shape, dtype, bias=False, accumulate=False, skew=0, most=2, seed=0):
    """The block with the identity as its gate on whole numbers: z and dz are whole numbers and every sum of products below
    2^24, so that z, and in fp32 every result, has to be equal; in 16 bits results are the sums rounded once."""
    n, d, f = shape
    rng = np.random.RandomState(seed + n + d + f)
    # (sparse: the sums of products stay small)
    x, w, b, dh = (whole_numbers(rng, s, most) * (rng.rand(*s) < 0.3) for s in ((n, d), (d, 2 * f), (2 * f,), (n, f)))
    b = b if bias else None
    z = x @ w + (0 if b is None else b)
    limit = {"f32": 2 ** 24, "bf16": 2 ** 8, "f16": 2 ** 11}[dtype]
    zk = np.clip(np.round(z), -2, 2)      # what the backward pass is given: any z
    dz, dx, dw, db = L.ff_backward(x, w, zk, dh, "none")
    sizes = np.abs(x) @ np.abs(w) + (0 if b is None else np.abs(b)), np.abs(dz) @ np.abs(w).T, np.abs(x).T @ np.abs(dz), np.abs(dz).sum(0)
    assert np.abs(dz).max() <= limit and max(v.max() for v in sizes) < 2 ** 24
    bx, bw, bdh = (Buf(T, v, dtype, skew) for v in (x, w, dh))
    bb = Buf(T, b, dtype, skew) if bias else None
    h, bz = out(T, (n, f), dtype, skew), out(T, (n, 2 * f), "f32", skew)
    T.gated_ff_fwd(d, f, bias, n, bx, bw, bb, h, bz, act="none", dtype=dtype)
    what = f"{dtype} batch {n} {d}->2*{f} skew {skew}"
    assert np.array_equal(bz.read(), z), what + " z"
    prod = z[:, :f] * z[:, f:]
    exact = np.abs(prod) < 2 ** 24
    L.within(h.read(), np.where(exact, L.rounded(prod, dtype), prod), np.where(exact, 0, (2.0 ** -23 + L.HALF_ULP[dtype]) * np.abs(prod)), what + " h")
    before = [whole_numbers(rng, s, 3) for s in ((d, 2 * f), (2 * f,))]
    bdx, bdw = out(T, (n, d), dtype, skew), Buf(T, before[0], dtype, skew)
    bdb = Buf(T, before[1], dtype, skew) if bias else None
    T.gated_ff_bwd(d, f, bias, n, bx, bw, Buf(T, zk, "f32", skew), bdh, bdx, bdw, bdb, act="none", dtype=dtype, accumulate=accumulate)
    add = 1 if accumulate else 0
    for got, want, name in ((bdx, dx, "dx"), (bdw, dw + add * before[0], "dw"), (bdb, db + add * before[1], "db")):
        if got is not None:
            L.within(got.read(), L.rounded(want, dtype), 0.0, what + " " + name)


@pytest.mark.parametrize("n", [5, 8])
@pytest.mark.parametrize("f", [1, 3])
def test_gated_ff_of_the_most_inputs(T, n, f):
    """(fp32: the weight gradient's tiles of rows, of which a launch takes 65535)"""
    ff_exact_case(T, (n, (1 << 21) - 1, f), "f32", bias=True)


# Sizes that are no multiple of anything, with which the three 16-bit products of a step come to each of the five tiles, with and without a
# split along the reduction (test_lm_plans.py holds them to that).
TILE_SHAPES = [(9, 9, 9), (11, 135, 11005), (1229, 3277, 9), (1327, 2291, 9), (383, 11, 5227), (63, 63, 91), (129, 11, 10931),
               (205, 275, 9979), (4225, 1409, 65), (3659, 3777, 165), (4541, 145, 2939), (65, 1361, 10405), (71, 8269, 1393),
               (5413, 391, 2801), (5509, 3385, 353)]


def name(shape):
    return "x".join(map(str, shape))


@pytest.mark.parametrize("dtype,aligned", [("bf16", False), ("f16", True), ("f16", False), ("bf16", True)])
@pytest.mark.parametrize("shape", TILE_SHAPES, ids=name)
def test_gated_ff_on_every_tile(T, shape, dtype, aligned):
    """(aligned: rows of whole 16-byte words, which are read where they lie; the others from padded copies)"""
    n, d, f = shape
    shape = (n, (d + 7) & ~7, (f + 7) & ~7) if aligned else shape
    ff_exact_case(T, shape, dtype, bias=True, accumulate=dtype == "f16")


FEW = [(1, 9000, 24), (2, 5000, 40), (3, 520, 1100), (4, 300, 70), (1, 64, 32), (1, 257, 100), (2, 8, 8), (3, 7, 33), (1, 1, 1), (4, 2111, 300),
       (2, 16411, 13)]
SOME = [(5, 100, 1), (7, 1, 64), (6, 64, 520), (8, 2100, 36), (17, 40, 24), (33, 128, 200), (65, 257, 130), (200, 320, 264)]
MANY = [(1001, 1024, 1000), (130, 2808, 2800), (3000, 264, 1400), (2000, 1208, 1224), (256, 1344, 1400), (2004, 1300, 1202), (402, 1401, 1803),
        (161, 1027, 2049), (67, 4097, 4099), (20001, 65, 801), (9001, 9, 5), (5000, 24, 40)]


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", FEW + SOME + MANY, ids=name)
def test_gated_ff_on_whole_numbers(T, shape, dtype):
    """No term of a sum is lost, or taken twice, however long it is."""
    ff_exact_case(T, shape, dtype, bias=True, accumulate=shape[0] % 2 == 0, skew=shape[0] % 3)


@pytest.mark.parametrize("dtype,n", [("f32", 1 << 20), ("bf16", (1 << 21) + 3), ("f16", (1 << 21) + 3)])
def test_gated_ff_of_the_most_samples_on_whole_numbers(T, dtype, n):
    ff_exact_case(T, (n, 1, 1), dtype, bias=True)
    ff_exact_case(T, (n, 3, 2), dtype, bias=True, accumulate=True)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4])
def test_gated_ff_of_a_few_rows_past_the_caches(T, n, dtype, accumulate):
    """(more than 32 MB of weights, at an odd length)"""
    ff_exact_case(T, (n, 2111, 4101), dtype, bias=True, accumulate=accumulate, skew=n % 2)


# ------------------------------------------------------------------ dropout

@pytest.mark.parametrize("residual", ["none", "apart", "in place"])
@pytest.mark.parametrize("dtype,n", [("f32", (1 << 23) + 5), ("bf16", (1 << 24) + 11), ("f16", (1 << 24) + 3)])
def test_dropout_past_the_caches(T, dtype, n, residual):
    """(more than 32 MB)"""
    rng = np.random.RandomState(7)
    x, r = (L.rounded(rng.randint(-64, 65, n), dtype) for _ in range(2))   # (halves and doubles of them are exact)
    keep = L.kept(n, 0.5, 3, 1 << 33)
    bx = Buf(T, x, dtype, 1)
    br = Buf(T, r, dtype, 1) if residual != "none" else None
    y = br if residual == "in place" else out(T, n, dtype, 1)
    T.dropout_seeded_fwd(n, bx, y, 0.5, 3, 1 << 33, residual=br, dtype=dtype)
    want = 2 * x * keep + (0 if br is None else r)
    assert np.array_equal(y.read(), L.rounded(want, dtype))
    T.dropout_seeded_bwd(n, bx, bx, 0.5, 3, 1 << 33, dtype=dtype)
    assert np.array_equal(bx.read(), 2 * x * keep)


# ------------------------------------------------------------------- losses

def logits(rows, vocab, dtype):
    rng = np.random.RandomState(rows + vocab)
    x = L.rounded(2 * rng.randn(rows, vocab), dtype)
    target = rng.randint(0, vocab, rows).astype(np.int32)
    target[rows // 2] = vocab - 1
    if rows > 3:
        target[1] = -1
    return x, target


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 3), (3, 300), (2, 9000), (3, 70001), (260, 40), (260, 700), (260, 9000), (257, 20011), (300, 33013)])
def test_token_logprob_alone(T, dtype, rows, vocab):
    """Without the statistics, as a reference model is scored: long rows are read past the caches then."""
    x, target = logits(rows, vocab, dtype)
    bx, bt, logp, twin, stats = Buf(T, x, dtype, 1), Buf(T, target, "i32"), out(T, rows), out(T, rows), out(T, (rows, 2))
    T.token_logprob_fwd(rows, vocab, bx, bt, logp, None, dtype=dtype)
    want = L.logprob(x, target)[0]
    L.within(logp.read(), want, L.lse_bound(x) + 2.0 ** -24 * np.abs(want), f"{dtype} {rows} rows of {vocab}")
    T.token_logprob_fwd(rows, vocab, bx, bt, twin, stats, dtype=dtype)
    assert np.array_equal(logp.bits(), twin.bits())


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [50, 9000, 33013])
@pytest.mark.parametrize("lengths", [[3, 2], [130, 0, 131, 5]], ids=str)
def test_preference_loss_alone(T, dtype, vocab, lengths):
    """Without a gradient."""
    rows, pairs = sum(lengths), len(lengths) // 2
    x, target = logits(rows, vocab, dtype)
    start = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    logp, sl, mg, loss = out(T, rows), out(T, 2 * pairs), out(T, pairs), out(T, 1)
    T.preference_loss(pairs, rows, vocab, Buf(T, x, dtype), Buf(T, target, "i32"), Buf(T, start, "i32"), None, logp, sl, mg, loss, None,
                      beta=0.25, dtype=dtype)
    now = L.logprob(x, target)[0]
    tol = L.lse_bound(x)
    L.within(logp.read(), now, tol + 2.0 ** -24 * np.abs(now), "logp")
    total = np.array([now[a:b].sum() for a, b in zip(start[:-1], start[1:])])
    seq_tol = tol * np.asarray(lengths) + 2.0 ** -40
    L.within(sl.read(), total, seq_tol + 2.0 ** -24 * np.abs(total), "sequences")
    m, pl, _ = L.preference(total, None, 0.25, 0.0, "sigmoid")
    m_tol = 0.25 * (seq_tol[0::2] + seq_tol[1::2])
    L.within(mg.read(), m, m_tol + 2.0 ** -24 * np.abs(m), "margins")
    L.within(loss.read(), [pl.mean()], m_tol.mean() + 2.0 ** -23 * pl.mean(), "loss")
