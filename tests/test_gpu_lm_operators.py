"""The language-model operators on the GPU against their definitions in 64 bits, at the sizes, types, alignments and
masks where they can go wrong. Bounds come from the number of roundings (lm_common.py)."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402

pytestmark = pytest.mark.gpu

CANARY = 0x5A


class Buf:
    """A device tensor of one of the types inside a larger allocation whose other bytes have to stay as they are.
    skew: elements that it starts behind a 256-byte boundary."""

    def __init__(self, T, values, dtype="f32", skew=0):
        self.T, self.dtype = T, dtype
        bits = values if dtype == "i32" else L.encode(values, dtype)
        self.shape, self.size = bits.shape, bits.dtype.itemsize
        self.lead = 256 + skew * self.size
        self.nbytes = bits.nbytes
        raw = np.full(self.lead + self.nbytes + 256, CANARY, np.uint8)
        raw[self.lead:self.lead + self.nbytes] = np.frombuffer(np.ascontiguousarray(bits).tobytes(), np.uint8)
        self.buf = T.DevBuf(raw.shape, np.uint8).upload(raw)
        self.ptr = T.DevBuf.view(self.buf.ptr.value + self.lead, self.shape, np.uint8).ptr

    def bits(self):
        raw = self.buf.numpy()
        assert (raw[:self.lead] == CANARY).all() and (raw[self.lead + self.nbytes:] == CANARY).all(), "written outside a tensor"
        kind = np.int32 if self.dtype == "i32" else L.NP[self.dtype]
        return np.frombuffer(raw[self.lead:self.lead + self.nbytes].tobytes(), kind).reshape(self.shape)

    def read(self):
        return L.decode(self.bits(), self.dtype)


def out(T, shape, dtype="f32", skew=0):
    return Buf(T, np.full(shape, 3.25), dtype, skew)


# ------------------------------------------------------------------ dropout

@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 17, 2047, 100003])
@pytest.mark.parametrize("skew", [0, 1])
def test_dropout(T, dtype, n, skew):
    rng = np.random.RandomState(n)
    x, dy, res = (L.rounded(rng.randn(n), dtype) for _ in range(3))
    seed, offset, rate = 0xFEDCBA9876543210, (1 << 40) + 3, 0.3
    keep = L.kept(n, rate, seed, offset)
    bx, bd, br = (Buf(T, v, dtype, skew) for v in (x, dy, res))
    y, y2, dx = (out(T, n, dtype, skew) for _ in range(3))
    T.dropout_seeded_fwd(n, bx, y, rate, seed, offset, dtype=dtype)
    T.dropout_seeded_fwd(n, bx, y2, rate, seed, offset, residual=br, dtype=dtype)
    T.dropout_seeded_bwd(n, bd, dx, rate, seed, offset, dtype=dtype)
    scale = 1.0 / (1.0 - np.float64(np.float32(rate)))
    # the factor and the product are rounded to fp32, the sum too, and the result to the type
    def bound(v):
        return 3 * 2.0 ** -24 * np.abs(v) + L.HALF_ULP[dtype] * np.abs(v) * (1 + 2.0 ** -20) + L.TINY[dtype]
    for got, want, extra in ((y, x * keep * scale, 0), (y2, x * keep * scale + res, 2.0 ** -22 * (np.abs(x) * scale)), (dx, dy * keep * scale, 0)):
        L.within(got.read(), want, bound(want) + extra, f"dropout {dtype} n={n}")
    assert (y.read()[~keep] == 0).all()


def test_dropout_masks_differ_by_offset_and_seed_and_repeat(T):
    n = 4096
    ones = Buf(T, np.ones(n))
    got = []
    for seed, offset in ((1, 0), (1, 1), (2, 0), (1, 1 << 32), (1 << 32, 0), (1, 0)):
        y = out(T, n)
        T.dropout_seeded_fwd(n, ones, y, 0.5, seed, offset)
        got.append(y.read() != 0)
        assert np.array_equal(got[-1], L.kept(n, 0.5, seed, offset))
    assert np.array_equal(got[0], got[-1])
    for i in range(5):
        for j in range(i):
            assert 0.4 < np.mean(got[i] == got[j]) < 0.6


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_dropout_in_place_rate_zero_and_exceptional_values(T, dtype):
    n = 1001
    x = np.random.RandomState(4).randn(n)
    x[5], x[6], x[7] = np.inf, -np.inf, np.nan
    x = L.rounded(x, dtype)
    b = Buf(T, x, dtype)
    T.dropout_seeded_fwd(n, b, b, 0.0, 9, 9, dtype=dtype)
    L.within(b.read(), x, 0.0, "rate 0 is the identity")
    keep = L.kept(n, 0.25, 9, 10)
    T.dropout_seeded_fwd(n, b, b, 0.25, 9, 10, dtype=dtype)
    want = np.where(keep, x, 0) * (1 / 0.75)  # what is dropped is zero, whatever it held
    L.within(b.read(), want, (3 * 2.0 ** -24 + L.HALF_ULP[dtype] * 1.001) * np.abs(np.where(np.isfinite(want), want, 0)) + L.TINY[dtype])
    res = Buf(T, np.ones(n), dtype)
    T.dropout_seeded_fwd(n, b, res, 0.25, 9, 11, residual=res, dtype=dtype)  # into the residual stream itself
    got = res.read()
    assert (got[~L.kept(n, 0.25, 9, 11)] == 1).all()
    T.dropout_seeded_fwd(0, b, b, 0.5, 1, dtype=dtype)


# ------------------------------------------------------- gated feed-forward

ACTS = ["silu", "gelu", "gelu_tanh", "sigmoid", "relu", "none"]
SHAPES = [(1, 1, 1), (1, 9000, 24), (2, 5000, 40), (3, 520, 1100), (4, 300, 70), (6, 64, 520), (8, 2100, 36), (9, 65, 40), (1, 64, 32), (1, 257, 100), (2, 8, 8), (3, 7, 33), (5, 100, 1), (7, 1, 64), (16, 64, 64), (17, 40, 24),
          (33, 128, 200), (64, 96, 128), (65, 257, 130), (130, 72, 72), (200, 320, 264)]


def ff_case(T, shape, act, dtype, bias, skew=0, accumulate=False, seed=0, scale=1.0):
    n, d, f = shape
    rng = np.random.RandomState(seed + n + 3 * d + 7 * f)
    x = L.rounded(scale * rng.randn(n, d), dtype)
    w = L.rounded(rng.randn(d, 2 * f) / np.sqrt(d), dtype)
    b = L.rounded(rng.randn(2 * f), dtype) if bias else None
    dh = L.rounded(rng.randn(n, f), dtype)
    bx, bw, bdh = (Buf(T, v, dtype, skew) for v in (x, w, dh))
    bb = Buf(T, b, dtype, skew) if bias else None
    h, h2, z = out(T, (n, f), dtype, skew), out(T, (n, f), dtype, skew), out(T, (n, 2 * f), "f32", skew)
    T.gated_ff_fwd(d, f, bias, n, bx, bw, bb, h, z, act=act, dtype=dtype)
    T.gated_ff_fwd(d, f, bias, n, bx, bw, bb, h2, None, act=act, dtype=dtype)
    what = f"{dtype} {act} batch {n} {d}->2*{f} skew {skew}"
    (zw, zb), (hw, hb) = L.ff_forward_bounds(x, w, b, act, dtype)
    L.within(z.read(), zw, zb, what + " z")
    L.within(h.read(), hw, hb, what + " h")
    L.within(h2.read(), hw, hb, what + " h without z")
    before = {k: L.rounded(rng.randn(*s), dtype) if accumulate else None for k, s in (("dw", (d, 2 * f)), ("db", (2 * f,)))}
    dx = out(T, (n, d), dtype, skew)
    dw = Buf(T, before["dw"], dtype, skew) if accumulate else out(T, (d, 2 * f), dtype, skew)
    db = None if not bias else Buf(T, before["db"], dtype, skew) if accumulate else out(T, (2 * f,), dtype, skew)
    T.gated_ff_bwd(d, f, bias, n, bx, bw, z, bdh, dx, dw, db, act=act, dtype=dtype, accumulate=accumulate)
    want = L.ff_backward_bounds(x, w, z.read(), dh, act, dtype)
    for k, got in (("dx", dx), ("dw", dw), ("db", db)):
        if got is None:
            continue
        v, e = want[k]
        if accumulate and k != "dx":
            v = v + before[k]
            e = e * (1 + 2.0 ** -20) + (L.HALF_ULP[dtype] + 2.0 ** -23) * np.abs(v) + 2.0 ** -23 * np.abs(before[k]) + L.TINY[dtype]
            if dtype != "f32":
                e = e + L.HALF_ULP[dtype] * np.abs(want[k][0])
        L.within(got.read(), v, e, what + " " + k)
    return (bx, bw, bb, z, bdh), (h, dx, dw, db)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gated_ff(T, dtype, shape):
    ff_case(T, shape, "silu", dtype, bias=shape[0] % 2 == 1)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", [(1001, 1024, 1000), (130, 2808, 2800), (700, 1336, 1200), (3000, 264, 1400), (300, 520, 392)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_ff_of_many_samples(T, dtype, shape):
    """(the largest tiles, products in three parts, sums split along k, last tiles that are shorter and narrower)"""
    ff_case(T, shape, "silu", dtype, bias=True)


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_gated_ff_of_many_samples_unaligned_and_accumulating(T, dtype):
    ff_case(T, (1001, 1024, 1000), "gelu", dtype, bias=True, skew=1, accumulate=True)


@pytest.mark.parametrize("shape", [(2000, 1208, 1224), (256, 1344, 1400), (2004, 1300, 1202)], ids=lambda s: "x".join(map(str, s)))
def test_gated_ff_of_many_samples_in_fours(T, shape):
    """(fp32: the weight gradient alone on planes, and all three products)"""
    ff_case(T, shape, "silu", "f32", bias=True)


@pytest.mark.parametrize("skew", [0, 1])
@pytest.mark.parametrize("shape", [(1001, 1027, 1001), (402, 1401, 1803), (130, 2811, 2797), (1500, 1340, 501), (20001, 65, 801), (161, 1027, 2049), (67, 4097, 4099)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_ff_of_many_samples_with_rows_of_any_length(T, shape, skew):
    """(fp32 products in three parts, whose copies are padded to whole words)"""
    ff_case(T, shape, "silu", "f32", bias=True, skew=skew, accumulate=skew == 1)


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_gated_ff_of_many_samples_with_infinities(T, dtype):
    """An infinite or NaN value reaches the sums that it is part of, which are what fp32 arithmetic gives, and no others."""
    many_samples_with_infinities(T, dtype, 1001, 1024, 1000)


@pytest.mark.parametrize("shape", [(1002, 1027, 1001), (1001, 1025, 505), (501, 1031, 1003)])
def test_gated_ff_of_many_samples_with_infinities_at_any_length(T, shape):
    many_samples_with_infinities(T, "f32", *shape)


def many_samples_with_infinities(T, dtype, n, d, f):
    rng = np.random.RandomState(12)
    x, w, dh = rng.randn(n, d), rng.randn(d, 2 * f) / 32, rng.randn(n, f)
    x[3, 17], x[n - 101, 5], x[n - 1, 1023] = np.inf, np.nan, -np.inf
    w[40, 7] = np.inf
    x, w, dh = (L.rounded(v, dtype) for v in (x, w, dh))
    bx, bw, bdh = (Buf(T, v, dtype) for v in (x, w, dh))
    h, z, dx, dw = out(T, (n, f), dtype), out(T, (n, 2 * f)), out(T, (n, d), dtype), out(T, (d, 2 * f), dtype)
    T.gated_ff_fwd(d, f, False, n, bx, bw, None, h, z, act="none", dtype=dtype)
    T.gated_ff_bwd(d, f, False, n, bx, bw, z, bdh, dx, dw, None, act="none", dtype=dtype)
    with np.errstate(all="ignore"):
        want = x @ w
        got = z.read()
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
        dz = L.rounded(np.concatenate([dh * got[:, f:], dh * got[:, :f]], 1), dtype)
        for g, v in ((dx.read(), dz @ w.T), (dw.read(), x.T @ dz)):
            assert np.array_equal(np.isfinite(g), np.isfinite(v)) and np.array_equal(np.isnan(g), np.isnan(v))


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gated_ff_activations(T, dtype, act):
    ff_case(T, (9, 48, 56), act, dtype, bias=True, scale=3.0)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n", [1, 9, 40])
def test_gated_ff_activations_far_from_zero(T, dtype, act, n):
    """Beyond 2^10 every activation is 0, 1 or the gate itself, and its derivative 0 or 1, without a rounding: squares and
    cubes that overflow on the way there must not show."""
    top = 15 if dtype == "f16" else 126
    g = np.array([s * 2.0 ** e for e in (10, 15, 30, 42, 63, 66, 90, 126) if e <= top for s in (1, -1)])
    f = len(g)
    want_h = {"sigmoid": (g > 0) * 1.0, "none": g}.get(act, np.maximum(g, 0))
    slope = {"sigmoid": 0 * g, "none": 0 * g + 1}.get(act, (g > 0) * 1.0)
    z = np.tile(np.concatenate([g, np.ones(f)]), (n, 1))
    x, w = Buf(T, np.ones((n, 1)), dtype), Buf(T, z[:1], dtype)
    h, bz = out(T, (n, f), dtype), out(T, (n, 2 * f))
    T.gated_ff_fwd(1, f, False, n, x, w, None, h, bz, act=act, dtype=dtype)
    assert np.array_equal(bz.read(), z) and np.array_equal(h.read(), np.tile(want_h, (n, 1)))
    db, dh = out(T, 2 * f, dtype), Buf(T, np.eye(n)[:, :1] * np.ones((n, f)), dtype)   # (one sample has a gradient)
    T.gated_ff_bwd(1, f, True, n, x, w, bz, dh, None, None, db, act=act, dtype=dtype)
    assert np.array_equal(db.read(), np.concatenate([slope, want_h]))


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", [(1, 64, 32), (6, 40, 48), (70, 64, 128)], ids=lambda s: "x".join(map(str, s)))
def test_gated_ff_unaligned_and_accumulating(T, dtype, shape):
    ff_case(T, shape, "gelu_tanh", dtype, bias=True, skew=1)
    ff_case(T, shape, "gelu_tanh", dtype, bias=True, accumulate=True)
    ff_case(T, shape, "gelu_tanh", dtype, bias=True, skew=3, accumulate=True)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("shape", [(513, 40, 48), (900, 41, 33), (5000, 24, 40), (9001, 9, 5), (4000, 1, 1)], ids=lambda s: "x".join(map(str, s)))
def test_gated_ff_of_many_samples_and_narrow_matrices(T, dtype, shape, accumulate):
    ff_case(T, shape, "silu", dtype, bias=True, accumulate=accumulate)


@pytest.mark.parametrize("dtype,n", [("f32", 1 << 20), ("bf16", (1 << 21) + 3)])
def test_gated_ff_of_the_most_samples(T, dtype, n):
    ff_case(T, (n, 1, 1), "sigmoid", dtype, bias=True)
    ff_case(T, (n, 3, 2), "sigmoid", dtype, bias=False)


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_gated_ff_gradients_left_out(T, dtype):
    """Each of dx, dw and db asked for alone. Another kernel may compute it then, in another order of its sums: two
    such sums are each within the bound of the definition's, so they are held to that and not to each other."""
    n, d, f = 37, 72, 88
    (x, w, b, z, dh), (_, dx, dw, db) = ff_case(T, (n, d, f), "silu", dtype, bias=True)
    want = L.ff_backward_bounds(x.read(), w.read(), z.read(), dh.read(), "silu", dtype)
    for k, whole in (("dx", dx), ("dw", dw), ("db", db)):
        one = out(T, whole.shape, dtype)
        T.gated_ff_bwd(d, f, True, n, x, w, z, dh, one if k == "dx" else None, one if k == "dw" else None,
                       one if k == "db" else None, act="silu", dtype=dtype)
        L.within(one.read(), *want[k], k + " alone")


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_gated_ff_without_rows(T, dtype):
    """The weight gradients of no samples are zero, or with accumulate what they were."""
    d, f = 9, 7
    x, w, h = (Buf(T, np.ones(s), dtype) for s in ((1, d), (d, 2 * f), (1, f)))
    z = Buf(T, np.ones((1, 2 * f)))
    dw, db = out(T, (d, 2 * f), dtype), out(T, 2 * f, dtype)
    T.gated_ff_fwd(d, f, False, 0, x, w, None, h, z, dtype=dtype)
    T.gated_ff_bwd(d, f, True, 0, x, w, z, h, x, dw, db, dtype=dtype, accumulate=True)
    assert (dw.read() == 3.25).all() and (db.read() == 3.25).all()
    T.gated_ff_bwd(d, f, True, 0, x, w, z, h, x, dw, db, dtype=dtype)
    assert (dw.read() == 0).all() and (db.read() == 0).all() and (h.read() == 1).all() and (x.read() == 1).all()


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_gated_ff_repeats_bit_for_bit(T, dtype):
    n, d, f = 130, 200, 104
    a, b = (ff_case(T, (n, d, f), "silu", dtype, bias=True)[1] for _ in range(2))
    for p, q in zip(a, b):
        assert np.array_equal(p.bits(), q.bits())


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("n", [1, 20, 150])
def test_gated_ff_exceptional_inputs_stay_in_their_rows(T, dtype, n):
    """NaN and infinities of one sample reach that sample's h and dx, and the sums over the batch; no other row."""
    d, f = 64, 72
    rng = np.random.RandomState(5)
    x, w, dh = rng.randn(n, d), rng.randn(d, 2 * f) / 8, rng.randn(n, f)
    x[n // 2, 3] = np.nan
    x[0, 5] = np.inf
    x, w, dh = (L.rounded(v, dtype) for v in (x, w, dh))
    bx, bw, bdh = (Buf(T, v, dtype) for v in (x, w, dh))
    h, z, dx, dw = out(T, (n, f), dtype), out(T, (n, 2 * f)), out(T, (n, d), dtype), out(T, (d, 2 * f), dtype)
    T.gated_ff_fwd(d, f, False, n, bx, bw, None, h, z, act="sigmoid", dtype=dtype)
    T.gated_ff_bwd(d, f, False, n, bx, bw, z, bdh, dx, dw, None, act="sigmoid", dtype=dtype)
    with np.errstate(all="ignore"):
        want = x @ w
    got = z.read()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
    rest = [r for r in range(n) if r not in (0, n // 2)]
    assert np.isfinite(h.read()[rest]).all() and np.isfinite(dx.read()[rest]).all()
    assert np.isnan(h.read()[n // 2]).all()


# ------------------------------------------------------------------- losses

VOCABS = [1, 2, 3, 10, 64, 257, 511, 1003, 2049, 8190, 16400, 33000, 70001, 131075]


def loss_inputs(rows, vocab, dtype, seed=0):
    rng = np.random.RandomState(seed + rows + vocab)
    x = L.rounded(2 * rng.randn(rows, vocab), dtype)
    target = rng.randint(0, vocab, rows).astype(np.int32)
    if rows > 2:
        target[1] = -1
        target[2] = vocab - 1
    return rng, x, target


def padded(x, ld, fill=7.5):
    """Rows ld elements apart, as one flat tensor that ends with the last row."""
    rows, vocab = x.shape
    flat = np.full((rows - 1) * ld + vocab, fill)
    for r in range(rows):
        flat[r * ld:r * ld + vocab] = x[r]
    return flat


def unpadded(flat, rows, vocab, ld):
    return np.stack([flat[r * ld:r * ld + vocab] for r in range(rows)])


def gaps(flat, rows, vocab, ld):
    keep = np.ones(len(flat), bool)
    for r in range(rows):
        keep[r * ld:r * ld + vocab] = False
    return flat[keep]


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_token_logprob(T, dtype, vocab):
    rows = 5
    for ld, skew in ((vocab, 0), (vocab + 3, 1)):
        rng, x, target = loss_inputs(rows, vocab, dtype)
        d = rng.randn(rows)
        d = L.rounded(d, "f32")
        bx, bt, bd = Buf(T, padded(x, ld), dtype, skew), Buf(T, target, "i32"), Buf(T, d)
        logp, stats, g = out(T, rows), out(T, (rows, 2)), Buf(T, padded(np.zeros((rows, vocab)), ld), dtype, skew)
        T.token_logprob_fwd(rows, vocab, bx, bt, logp, stats, dtype=dtype, ld=ld)
        T.token_logprob_bwd(rows, vocab, bx, bt, stats, bd, g, dtype=dtype, ld=ld, ld_d=ld)
        want_logp, want_stats, _, _ = L.logprob(x, target)
        tol = L.lse_bound(x)
        what = f"{dtype} vocab {vocab} ld {ld}"
        L.within(stats.read(), want_stats, np.stack([np.zeros(rows), (tol + 2.0 ** -24) * want_stats[:, 1]], 1), what)
        L.within(logp.read(), want_logp, tol + 2.0 ** -24 * np.abs(want_logp), what)
        flat = g.read()
        L.within(unpadded(flat, rows, vocab, ld), L.dlogits(x, target, d),
                 L.dlogits_bound(x, target, d, np.zeros(rows), dtype), what + " gradient")
        assert (gaps(flat, rows, vocab, ld) == 7.5).all(), "written between rows"
        # in the logits' place, and with rows of the gradient at another distance than the logits'
        other = Buf(T, padded(np.zeros((rows, vocab)), vocab + 1), dtype, skew + 1)
        T.token_logprob_bwd(rows, vocab, bx, bt, stats, bd, other, dtype=dtype, ld=ld, ld_d=vocab + 1)
        assert np.array_equal(unpadded(other.read(), rows, vocab, vocab + 1), unpadded(flat, rows, vocab, ld))
        T.token_logprob_bwd(rows, vocab, bx, bt, stats, bd, bx, dtype=dtype, ld=ld, ld_d=ld)
        assert np.array_equal(unpadded(bx.read(), rows, vocab, ld), unpadded(flat, rows, vocab, ld))


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [5, 300, 5000, 140000])
def test_token_logprob_exceptional_rows(T, dtype, vocab):
    """Masks of -inf and of the type's lowest value, a row with nothing left, infinities, NaN, targets past the
    end, and NaN in rows that do not count."""
    lowest = {"f32": -np.finfo(np.float32).max, "bf16": L.decode(np.uint16([0xFF7F]), "bf16")[0], "f16": -65504.0}[dtype]
    rng = np.random.RandomState(6)
    x = L.rounded(rng.randn(10, vocab), dtype)
    target = np.zeros(10, np.int32)
    x[0, 1:] = -np.inf              # one token is left
    x[1, 1:] = lowest
    x[2, :] = -np.inf               # nothing is left
    x[3, :] = lowest                # all equally unlikely
    x[4, 2] = np.inf
    x[5, 2] = np.nan
    x[6, :], target[6] = np.nan, -1  # padding
    target[7] = vocab
    target[8] = np.iinfo(np.int32).max
    x[9, 0] = -np.inf               # the token itself is masked
    d = L.rounded(rng.randn(10), "f32")
    bx, bt, bd = Buf(T, x, dtype), Buf(T, target, "i32"), Buf(T, d)
    logp, stats, g = out(T, 10), out(T, (10, 2)), out(T, (10, vocab), dtype)
    T.token_logprob_fwd(10, vocab, bx, bt, logp, stats, dtype=dtype)
    T.token_logprob_bwd(10, vocab, bx, bt, stats, bd, g, dtype=dtype)
    got, gs, gg = logp.read(), stats.read(), g.read()
    tol = L.lse_bound(x)
    assert got[0] == 0 and gs[0, 0] == x[0, 0] and gs[0, 1] == 1 and abs(got[1]) <= tol
    assert np.isnan(got[2]) and gs[2, 0] == -np.inf and np.isnan(gg[2]).all()
    assert abs(got[3] + np.log(vocab)) <= tol + 2.0 ** -24 * np.log(vocab) and gs[3, 0] == lowest
    assert np.isnan(got[4]) and np.isnan(got[5]) and np.isnan(gg[5]).all()
    assert got[6] == 0 and (gs[6] == 0).all() and (gg[6] == 0).all()
    assert np.isnan(got[7:9]).all() and np.isnan(gg[7:9]).all()
    assert got[9] == -np.inf and np.isfinite(gg[9]).all()
    assert (gg[0] == 0).all()
    for r in (1, 3, 9):
        want = L.dlogits(x[r:r + 1], target[r:r + 1], d[r:r + 1])
        L.within(gg[r:r + 1], want, L.dlogits_bound(x[r:r + 1], target[r:r + 1], d[r:r + 1], np.zeros(1), dtype))


def policy_case(T, dtype, rows, vocab, ld, skew, use_ref, use_weight, in_place):
    low, high, kl = 0.2, 0.3, 0.07
    rng, x, target = loss_inputs(rows, vocab, dtype, 1)
    now = L.logprob(x, target)[0]
    old, ref = L.rounded(now + 0.3 * rng.randn(rows), "f32"), L.rounded(now + 0.5 * rng.randn(rows), "f32")
    adv, weight = L.rounded(rng.randn(rows), "f32"), L.rounded(rng.rand(rows), "f32")
    low, high, kl = (float(np.float32(v)) for v in (low, high, kl))
    # (no row so near a clipping bound that rounding decides on which side of it it falls)
    near = (np.abs(np.exp(now - old)[:, None] - [1 - low, 1 + high]) < 1e-3).any(1)
    old = L.rounded(np.where(near, old + 0.01, old), "f32")
    bx, bt = Buf(T, padded(x, ld), dtype, skew), Buf(T, target, "i32")
    g = bx if in_place else Buf(T, padded(np.zeros((rows, vocab)), ld), dtype, skew)
    logp, row, total = out(T, rows), out(T, rows), out(T, 1)
    T.policy_loss(rows, vocab, bx, bt, Buf(T, old), Buf(T, ref) if use_ref else None, Buf(T, adv),
                  Buf(T, weight) if use_weight else None, logp, row, total, g, clip_low=low, clip_high=high, kl_coef=kl,
                  dtype=dtype, ld=ld, ld_d=ld)
    w = weight if use_weight else None
    want_row, d = L.policy(now, target, old, ref if use_ref else None, adv, w, low, high, kl)
    what = f"policy {dtype} {rows}x{vocab}"
    tol = L.lse_bound(x)
    L.within(logp.read(), now, tol + 2.0 ** -24 * np.abs(now), what)
    # the loss and d change with logp by no more than |w| (ratio |adv| + kl (1 + exp(gap)))
    slope = (weight if use_weight else 1) * (np.exp(now - old) * np.abs(adv) + kl * (1 + np.exp(ref - now))) * 1.01
    # a row within the ratio's error (at most 1.31 of tol next to the bounds) of a clipping bound may fall on either
    # side of it: there is none in these inputs
    ratio = np.exp(now - old)
    assert np.min(np.abs(ratio[target >= 0][:, None] - [1 - low, 1 + high])) > 2 * tol
    L.within(row.read(), want_row, slope * tol + 2.0 ** -24 * np.abs(want_row), what)
    L.within(total.read(), [want_row.sum()], slope.sum() * tol + 2.0 ** -23 * np.abs(want_row).sum(), what)
    flat = g.read()
    L.within(unpadded(flat, rows, vocab, ld), L.dlogits(x, target, d),
             L.dlogits_bound(x, target, d, slope * tol + 2.0 ** -24 * np.abs(d), dtype), what + " gradient")
    assert (gaps(flat, rows, vocab, ld) == 7.5).all()


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_policy_loss(T, dtype, vocab):
    policy_case(T, dtype, 6, vocab, vocab, 0, True, True, False)
    policy_case(T, dtype, 5, vocab, vocab + 5, 1, False, False, True)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [33, 700, 3000, 9000, 20000])
def test_losses_of_more_rows_than_compute_units(T, dtype, vocab):
    """(where a row has fewer waves)"""
    policy_case(T, dtype, 260, vocab, vocab, 0, True, True, False)
    preference_case(T, dtype, [130, 133], vocab, "sigmoid", 0.1, vocab, 0, True)


@pytest.mark.parametrize("rows", [1, 4, 5, 100, 1024, 1025, 1500])
def test_policy_loss_rows(T, rows):
    policy_case(T, "f32", rows, 10, 10, 0, True, True, False)
    policy_case(T, "bf16", rows, 37, 40, 0, True, False, False)


def test_policy_loss_outputs_left_out_and_no_rows(T):
    rng, x, target = loss_inputs(9, 50, "f32")
    bx, bt, v = Buf(T, x), Buf(T, target, "i32"), Buf(T, rng.randn(9))
    a, b, total, only = out(T, 9), out(T, 9), out(T, 1), out(T, 1)
    g, g2 = out(T, (9, 50)), out(T, (9, 50))
    T.policy_loss(9, 50, bx, bt, v, v, v, None, a, b, total, g, kl_coef=0.1)
    T.policy_loss(9, 50, bx, bt, v, v, v, None, None, None, only, None, kl_coef=0.1)
    T.policy_loss(9, 50, bx, bt, v, v, v, None, None, None, None, g2, kl_coef=0.1)
    assert np.array_equal(total.bits(), only.bits()) and np.array_equal(g.bits(), g2.bits())
    T.policy_loss(0, 50, bx, bt, v, v, v, None, None, None, only, None)
    assert only.read()[0] == 0
    none = Buf(T, np.full(9, -1, np.int32), "i32")
    T.policy_loss(9, 50, bx, none, v, v, v, None, a, b, only, g)
    assert only.read()[0] == 0 and (a.read() == 0).all() and (b.read() == 0).all() and (g.read() == 0).all()


def test_policy_loss_on_the_bound(T):
    """Equal sides of the minimum (the policy as it was: ratio 1, bounds 1) take the free side's gradient; a ratio past
    the bound on the side that the advantage does not reward keeps it."""
    x = np.zeros((4, 2))
    target = np.zeros(4, np.int32)
    now = -np.log(2.0)
    old = L.rounded(np.array([now, now, now - 1, now + 1]), "f32")
    adv = np.array([1.0, -1.0, -1.0, 1.0])
    bx, g, row = Buf(T, x), out(T, (4, 2)), out(T, 4)
    T.policy_loss(4, 2, bx, Buf(T, target, "i32"), Buf(T, old), None, Buf(T, adv), None, None, row, None, g, clip_low=0.5,
                  clip_high=0.5)
    r = np.exp(now - old)
    L.within(row.read(), -r * adv, 2.0 ** -20)
    L.within(g.read(), np.stack([-r * adv / 2, r * adv / 2], 1), 2.0 ** -20)


def preference_case(T, dtype, lengths, vocab, kind, smoothing, ld, skew, use_ref, lead=0, trail=0, in_place=False):
    beta = float(np.float32(0.3))
    smoothing = float(np.float32(smoothing))
    pairs = len(lengths) // 2
    start = (lead + np.concatenate([[0], np.cumsum(lengths)])).astype(np.int32)
    rows = int(start[-1]) + trail
    rng, x, target = loss_inputs(rows, vocab, dtype, 2)
    now = L.logprob(x, target)[0]
    inside = (np.arange(rows) >= start[0]) & (np.arange(rows) < start[-1])
    seq = np.clip(np.searchsorted(start, np.arange(rows), side="right") - 1, 0, 2 * pairs - 1)
    total = np.bincount(seq[inside], now[inside], minlength=2 * pairs)
    ref = L.rounded(total + rng.randn(2 * pairs), "f32")
    bx = Buf(T, padded(x, ld), dtype, skew)
    g = bx if in_place else Buf(T, padded(np.full((rows, vocab), 2.5), ld), dtype, skew)
    logp, sl, mg, loss = out(T, rows), out(T, 2 * pairs), out(T, pairs), out(T, 1)
    T.preference_loss(pairs, rows, vocab, bx, Buf(T, target, "i32"), Buf(T, start, "i32"), Buf(T, ref) if use_ref else None, logp,
                      sl, mg, loss, g, beta=beta, smoothing=smoothing, kind=kind, dtype=dtype, ld=ld, ld_d=ld)
    m, pl, d = L.preference(total, ref if use_ref else None, beta, smoothing, kind)
    what = f"preference {dtype} {kind} vocab {vocab}"
    tol = L.lse_bound(x)
    L.within(logp.read()[inside], now[inside], tol + 2.0 ** -24 * np.abs(now[inside]), what)
    assert (logp.read()[~inside] == 3.25).all()
    seq_tol = tol * np.asarray(lengths) + 2.0 ** -40
    L.within(sl.read(), total, seq_tol + 2.0 ** -24 * np.abs(total), what)
    m_tol = beta * (seq_tol[0::2] + seq_tol[1::2])
    L.within(mg.read(), m, m_tol + 2.0 ** -23 * np.abs(m), what)
    steep = {"sigmoid": 1.0, "hinge": 1.0, "squared": 2 * (np.max(np.abs(m)) + 1) / beta ** 2}[kind]
    L.within(loss.read(), [pl.mean()], steep * m_tol.mean() + 2.0 ** -23 * np.abs(pl).mean(), what)
    if kind == "hinge":
        assert np.min(np.abs(m - 1)) > 10 * np.max(m_tol)
    curve = {"sigmoid": 0.25, "hinge": 0.0, "squared": 2 / beta ** 2}[kind]
    d_off = np.repeat(beta * curve * m_tol / pairs, 2) + 2.0 ** -23 * np.abs(d)
    flat = g.read()
    got = unpadded(flat, rows, vocab, ld)
    L.within(got[inside], L.dlogits(x, target, d[seq])[inside], L.dlogits_bound(x, target, d[seq], d_off[seq], dtype)[inside],
             what + " gradient")
    assert np.array_equal(got[~inside], x[~inside] if in_place else np.full_like(got[~inside], 2.5)), "rows outside the sequences"
    assert (gaps(flat, rows, vocab, ld) == 7.5).all()


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("squared", 0.0), ("hinge", 0.0)])
def test_preference_loss(T, dtype, kind, smoothing):
    preference_case(T, dtype, [4, 7, 1, 3], 33, kind, smoothing, 33, 0, True)
    preference_case(T, dtype, [9, 2], 1003, kind, smoothing, 1010, 1, False, lead=2, trail=3)
    preference_case(T, dtype, [0, 5, 3, 0, 0, 0], 40, kind, smoothing, 40, 0, True, trail=1)


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [1, 5, 9000, 70001])
def test_preference_loss_vocabularies(T, dtype, vocab):
    preference_case(T, dtype, [3, 2, 2, 4], vocab, "sigmoid", 0.0, vocab, 0, True, in_place=True, lead=1, trail=1)


def test_preference_loss_long_and_many(T):
    preference_case(T, "f32", [700, 513], 11, "sigmoid", 0.05, 11, 0, True)
    preference_case(T, "bf16", list(np.random.RandomState(8).randint(0, 9, 300)), 17, "sigmoid", 0.0, 17, 0, True)


@pytest.mark.parametrize("kind", ["sigmoid", "squared", "hinge"])
def test_preference_loss_with_and_without_a_launch_for_the_pairs(T, kind):
    preference_case(T, "f32", [600, 400], 50, kind, 0.0, 50, 0, True)
    preference_case(T, "bf16", [3, 4, 0, 65, 2, 1, 9, 9, 1, 0, 5, 6, 7, 8, 64, 63], 1200, kind, 0.0, 1201, 0, False, lead=1, trail=2)
    preference_case(T, "bf16", [3, 4, 0, 65, 2, 1, 9, 9, 1, 0, 5, 6, 7, 8, 64, 63, 2, 2], 1200, kind, 0.0, 1201, 0, False, lead=1, trail=2)


def test_preference_loss_without_pairs_rows_or_outputs(T):
    loss = out(T, 1)
    i32 = Buf(T, np.zeros(5, np.int32), "i32")
    x = Buf(T, np.zeros((3, 4)))
    T.preference_loss(0, 3, 4, x, i32, None, loss=loss)
    assert loss.read()[0] == 0
    m = out(T, 2)
    T.preference_loss(2, 0, 4, x, i32, i32, margin=m, loss=loss)   # two pairs of empty sequences
    assert (m.read() == 0).all() and abs(loss.read()[0] - np.log(2)) < 1e-7
    T.preference_loss(1, 3, 4, x, i32, Buf(T, np.array([0, 2, 3], np.int32), "i32"))


def test_preference_large_margins_do_not_overflow(T):
    """Margins of thousands: the loss is linear, the gradient saturates."""
    x = np.zeros((2, 2))
    x[0, 0], x[1, 0] = 20000.0, -20000.0
    for t, want in (([0, 0], 0.0), ([1, 1], 20000.0)):
        loss, g = out(T, 1), out(T, (2, 2))
        T.preference_loss(1, 2, 2, Buf(T, x), Buf(T, np.array(t, np.int32), "i32"), Buf(T, np.array([0, 1, 2], np.int32), "i32"),
                          loss=loss, dlogits=g, beta=1.0)
        assert abs(loss.read()[0] - want) <= 1e-3 and np.isfinite(g.read()).all()


# -------------------------------------------------------------------- casts

def test_cast(T):
    rng = np.random.RandomState(9)
    v = np.concatenate([rng.randn(1000) * 10.0 ** rng.randint(-12, 12, 1000), [0, -0.0, np.inf, -np.inf, np.nan, 1e-40, 65519, 65520]])
    v = L.rounded(v, "f32")
    for src in L.DTYPES:
        for dst in L.DTYPES:
            with np.errstate(over="ignore"):
                a = L.rounded(v, src)
                want = L.rounded(a, dst)
            o = out(T, len(v), dst)
            T.cast(len(v), Buf(T, a, src), o, src, dst)
            L.within(o.read(), want, 0.0, f"{src} -> {dst}")


# ------------------------------------------------- a step made of the operators

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_training_step_of_the_operators_together(T, dtype):
    """Block, dropout into the residual stream, logits by a fully-connected layer (fp32), policy loss, and the way
    back to the block's weights and their update: against the same in 64 bits, and against differences of the loss."""
    n, d, f, v, seed = 24, 32, 48, 19, 11
    rng = np.random.RandomState(7)
    q = lambda a: L.rounded(a, dtype)  # noqa: E731
    x, w1, b1 = q(rng.randn(n, d)), q(rng.randn(d, 2 * f) / 6), q(0.1 * rng.randn(2 * f))
    w2, b2, w3 = L.rounded(rng.randn(f, d) / 7, "f32"), L.rounded(0.1 * rng.randn(d), "f32"), L.rounded(rng.randn(d, v) / 3, "f32")
    target = rng.randint(0, v, n).astype(np.int32)
    target[3] = -1
    adv = L.rounded(rng.randn(n), "f32")
    rate, scale = 0.25, 1 / 0.75
    keep = L.kept(n * d, rate, seed, 2).reshape(n, d)

    def forward(x, w1, b1):
        z, h = L.ff_forward(x, w1, b1, "silu")
        y = x + (h @ w2 + b2) * keep * scale
        return z, h, y, y @ w3

    z, h, y, logits = forward(x, w1, b1)
    now = L.logprob(logits, target)[0]
    old, ref = L.rounded(now + 0.05 * rng.randn(n), "f32"), L.rounded(now + 0.2 * rng.randn(n), "f32")

    def loss_of(x, w1, b1):
        return L.policy(L.logprob(forward(x, w1, b1)[3], target)[0], target, old, ref, adv, None, 0.2, 0.2, 0.1)[0].sum()

    bx, bw1, bb1 = Buf(T, x, dtype), Buf(T, w1, dtype), Buf(T, b1, dtype)
    bw2, bb2, bw3 = Buf(T, w2), Buf(T, b2), Buf(T, w3)
    bz, bh, hf, o, xf = out(T, (n, 2 * f)), out(T, (n, f), dtype), out(T, (n, f)), out(T, (n, d)), out(T, (n, d))
    by, bl, total, g = out(T, (n, d)), out(T, (n, v)), out(T, 1), out(T, (n, v))
    T.gated_ff_fwd(d, f, True, n, bx, bw1, bb1, bh, bz, act="silu", dtype=dtype)
    if dtype == "f32":
        hf, xf = bh, bx
    else:
        T.cast(n * f, bh, hf, dtype, "f32")
        T.cast(n * d, bx, xf, dtype, "f32")
    T.fc_fwd(f, d, True, n, hf, bw2, bb2, o)
    T.dropout_seeded_fwd(n * d, o, by, rate, seed, 2, residual=xf)
    T.fc_fwd(d, v, False, n, by, bw3, None, bl)
    T.policy_loss(n, v, bl, Buf(T, target, "i32"), Buf(T, old), Buf(T, ref), Buf(T, adv), None, None, None, total, g, kl_coef=0.1)
    dy, do, dh, dw1, db1, dx = out(T, (n, d)), out(T, (n, d)), out(T, (n, f)), out(T, (d, 2 * f), dtype), out(T, 2 * f, dtype), out(T, (n, d), dtype)
    T.fc_bwd(d, v, False, n, by, bw3, g, dy, None, None)
    T.dropout_seeded_bwd(n * d, dy, do, rate, seed, 2)
    T.fc_bwd(f, d, True, n, hf, bw2, do, dh, None, None)
    dht = dh
    if dtype != "f32":
        dht = out(T, (n, f), dtype)
        T.cast(n * f, dh, dht, "f32", dtype)
    T.gated_ff_bwd(d, f, True, n, bx, bw1, bz, dht, dx, dw1, db1, act="silu", dtype=dtype)
    grad = dw1
    if dtype != "f32":
        grad = out(T, (d, 2 * f))
        T.cast(2 * d * f, dw1, grad, dtype, "f32")
    weights = Buf(T, w1)
    T.opt_update(T.opt_desc("sgd", alpha=0.5), 2 * d * f, grad, weights)
    # in 64 bits
    dl = L.dlogits(logits, target, L.policy(now, target, old, ref, adv, None, 0.2, 0.2, 0.1)[1])
    ddy = dl @ w3.T
    ddh = (ddy * keep * scale) @ w2.T
    _, ddx, ddw, ddb = L.ff_backward(x, w1, z, ddh, "silu")
    # in fp32 sums of some fifty products each; in bf16 h, dh, dz and the results are rounded (half a step of 2^-8 each)
    rel = 2.0 ** -16 if dtype == "f32" else 6 * 2.0 ** -8
    for got, want, what in ((total.read(), [loss_of(x, w1, b1)], "loss"), (dw1.read(), ddw, "dw"), (db1.read(), ddb, "db"),
                            (dx.read(), ddx, "dx"), (weights.read(), w1 - 0.5 * ddw, "updated weights")):
        want = np.asarray(want)
        size = np.abs(want).max() if what != "loss" else np.abs(adv).sum()
        L.within(got, want, rel * size, what)
    for i in ((0, 0), (5, 50), (31, 95)):   # the gradient's chain in 64 bits against differences
        e = np.zeros_like(w1)
        e[i] = 1e-6
        assert abs((loss_of(x, w1 + e, b1) - loss_of(x, w1 - e, b1)) / 2e-6 - ddw[i]) < 1e-5 * (1 + abs(ddw[i]))


# --------------------------------------- dropout layers that draw for themselves

def dropout_net(T, flags, batch, rng):
    """fc - tanh - dropout - fc - dropout - fc under mse, with set weights"""
    net = T.Net([T.L_fc(12, 37), T.L_act("tanh"), T.L_dropout(0.3), T.L_fc(37, 21), T.L_dropout(0.6), T.L_fc(21, 5)], batch, flags)
    for i, which, n in net.params():
        net.set_param(i, which, (rng.randn(n) / 4).astype(np.float32))
    return net


def check_dropout_step(net, batch, seeds, p):
    """Both dropout layers of the last step against the masks of pass p, forward and backward."""
    for layer, rate in ((2, 0.3), (4, 0.6)):
        n = batch * net.layer_out_size(layer)
        keep = L.kept(n, rate, *[seeds[layer][0], seeds[layer][1] + p]).reshape(batch, -1)
        scale = 1 / (1 - np.float64(np.float32(rate)))
        x, y = net.layer_out(layer - 1, batch), net.layer_out(layer, batch)
        L.within(y, x.astype(np.float64) * keep * scale, 2.0 ** -22 * np.abs(x) * scale, f"layer {layer}, pass {p}")
        dy, dx = net.layer_dx(layer + 1, batch), net.layer_dx(layer, batch)
        L.within(dx, dy.astype(np.float64) * keep * scale, 2.0 ** -22 * np.abs(dy) * scale, f"layer {layer}, pass {p}, backward")


@pytest.mark.parametrize("flags", [0, 1, 2, 3, 7])
def test_net_draws_its_dropout_masks(T, flags):
    """Another mask every pass, with and without a captured step (each of them replayed, with other work between the
    replays); several steps a call are the single steps; the test phase is the identity and draws nothing; a mask
    that is handed over takes the generator's place until the next one is set."""
    batch, rng = 9, np.random.RandomState(3)
    x, t = T.to_device(rng.randn(batch, 12)), T.to_device(rng.randn(batch, 5))
    seeds = {2: (77, 1000), 4: (1 << 63, 0)}
    net, twin = dropout_net(T, flags, batch, np.random.RandomState(4)), dropout_net(T, 0, batch, np.random.RandomState(4))
    opt, topt = T.opt_desc("momentum"), T.opt_desc("momentum")
    with pytest.raises(T.TdhError, match="one step a call"):
        net.train_steps(opt, "mse", batch, [x, x], [t, t])
    for n in (net, twin):
        for layer, (seed, offset) in seeds.items():
            n.set_dropout_generator(layer, seed, offset)
    for p in range(5):
        net.train_step(opt, "mse", batch, x, t)
        check_dropout_step(net, batch, seeds, p)
        T.sync()
        T.fill_zero(T.DevBuf(1000))
    net.forward(batch, x)                      # pass 5
    keep = L.kept(batch * 37, 0.3, 77, 1005).reshape(batch, -1)
    assert np.array_equal(net.layer_out(2, batch) != 0, keep)
    net.set_phase(False)
    net.forward(batch, x)
    assert np.array_equal(net.layer_out(2, batch), net.layer_out(1, batch))
    net.set_phase(True)
    net.train_steps(opt, "mse", batch, [x] * 4, [t] * 4)   # passes 6 to 9
    check_dropout_step(net, batch, seeds, 9)
    net.train_steps(opt, "mse", batch, [x] * 4, [t] * 4)   # and 10 to 13, the same graph again
    check_dropout_step(net, batch, seeds, 13)
    for p in range(14):
        if p == 5:
            twin.forward(batch, x)
        else:
            twin.train_step(topt, "mse", batch, x, t)
    for i, which, _ in net.params():
        L.within(net.get_param(i, which), twin.get_param(i, which), 2e-6 if flags else 0.0, f"parameter {i}.{which}")
    mask = np.ones((batch, 37), np.uint8)
    net.set_dropout_mask(2, mask)
    net.train_step(opt, "mse", batch, x, t)
    a, b = net.layer_out(1, batch), net.layer_out(2, batch)
    L.within(b, a / (1 - 0.3), 2.0 ** -21 * np.abs(a), "a mask that was handed over")
    with pytest.raises(T.TdhError, match="one step a call"):
        net.train_steps(opt, "mse", batch, [x, x], [t, t])
    net.set_dropout_generator(2, 77, 0)
    net.train_step(opt, "mse", batch, x, t)
    assert np.array_equal(net.layer_out(2, batch) != 0, L.kept(batch * 37, 0.3, 77, 0).reshape(batch, -1))
    with pytest.raises(T.TdhError):
        net.set_dropout_generator(1, 77)       # not a dropout layer
    with pytest.raises(T.TdhError):
        net.set_dropout_generator(6, 77)
    net.close()
    twin.close()


def test_gradient_of_a_net_that_draws_its_dropout_masks(T):
    """Against differences of its own loss, the mask held by setting the same offset again."""
    batch, rng = 6, np.random.RandomState(8)
    x, t = T.to_device(rng.randn(batch, 12)), rng.randn(batch, 5)
    net = dropout_net(T, 0, batch, np.random.RandomState(9))

    def again():
        net.set_dropout_generator(2, 5, 50)
        net.set_dropout_generator(4, 6, 60)

    def loss():
        again()
        net.forward(batch, x)
        return np.sum((net.layer_out(5, batch).astype(np.float64) - t) ** 2) / 5   # mse::df is 2 (y - t) / n

    again()
    net.train_step(None, "mse", batch, x, T.to_device(t), do_update=False)
    for i, which, n in net.params():
        grad, w = net.layer_grad(i, which), net.get_param(i, which)
        for k in (0, n // 2, n - 1):
            e = np.zeros(n, np.float32)
            e[k] = 2.0 ** -6
            net.set_param(i, which, w + e)
            up = loss()
            net.set_param(i, which, w - e)
            down = loss()
            net.set_param(i, which, w)
            # third derivatives times (2^-6)^2 / 6, and fp32 outputs of order 1
            assert abs((up - down) * 32 - grad[k]) < 2e-3 * (1 + abs(grad[k])), (i, which, k)
    net.close()
