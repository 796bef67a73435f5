"""Tokens drawn from logits on the GPU: the token itself, the number left and both log-probabilities against the definition in 64 bits."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, kept, logp, logq) of one row, and how far u is from the next border."""
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return -1, 0, np.nan, np.nan, 1.0
    if not temperature > 0:
        temperature, top_k, top_p, min_p = 1.0, 1, 1.0, 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        t = np.where(x[order] == x[order[0]], 0.0, (x[order] - x[order[0]]) / temperature)
    w = np.exp(t)
    margin = 1.0
    if top_p < 1:
        cum = np.cumsum(w)
        n = int(np.argmax(cum >= max(top_p, 0.0) * cum[-1])) + 1
        margin = np.min(np.abs(cum[max(0, n - 2):n + 1] / cum[-1] - top_p))
        order, w, t = order[:n], w[:n], t[:n]
    n = max(1, int((w >= min(min_p, 1.0)).sum())) if min_p > 0 else len(w)
    order, w, t = order[:n], w[:n], t[:n]
    by_index = np.argsort(order)
    cum = np.cumsum(w[by_index])
    u = 0.0 if not u > 0 else min(float(u), np.nextafter(1.0, 0))
    at = min(int((cum <= u * cum[-1]).sum()), n - 1)
    while w[by_index[at]] == 0:   # (the last one that weighs anything)
        at -= 1
    margin = min(margin, np.min(np.abs(cum / cum[-1] - u)) if n > 1 else 1.0)
    chosen = order[by_index[at]]
    d = np.delete(x[x > -np.inf], np.argmax(x[x > -np.inf])) - x.max()
    log1 = lambda v: np.log1p(np.sum(v))  # noqa: E731
    return chosen, n, x[chosen] - x.max() - log1(np.exp(d)), t[by_index[at]] - log1(w[1:]), margin


def run(T, x, u, dtype, settings=None, skew=0, ld=None, **kw):
    rows = len(u)
    vocab = x.shape[1] if ld is None else kw.pop("vocab")
    bx, bu = Buf(T, x, dtype, skew), Buf(T, u)
    tok, kept = (Buf(T, np.full(rows, 77, np.int32), "i32") for _ in range(2))
    logp, logq = out(T, rows), out(T, rows)
    s = None
    if settings is not None:
        raw = np.zeros((rows, 4), np.int32)
        for i, c in enumerate(settings):
            raw[i, [0, 2, 3]] = np.array([c[0], c[2], c[3]], np.float32).view(np.int32)
            raw[i, 1] = c[1]
        s = Buf(T, raw, "i32")
    T.sample_tokens(rows, vocab, bx, bu, tok, logp, logq, kept, settings=s, dtype=dtype, ld=ld, **kw)
    return tok.bits(), kept.bits(), logp.read(), logq.read()


def f32(v):
    return float(np.float32(v))


def check(T, x, u, dtype, settings, got, what=""):
    for i in range(len(u)):
        t, k, p, q = settings[i]
        token, kept, logp, logq, margin = draw(x[i], u[i], f32(t), k, f32(p), f32(q))
        # the sums are off by 2^-46 a token, and so are the double sums here
        if margin < 1e-9:
            continue
        assert got[0][i] == token, (what, i, settings[i], got[0][i], token)
        assert got[1][i] == kept, (what, i, settings[i], got[1][i], kept)
        for g, w in ((got[2][i], logp), (got[3][i], logq)):
            if np.isnan(w):
                assert np.isnan(g)
            else:
                # one rounding of the result (below fp32's smallest number, 2^-149, to a multiple of that: half of it off at most, 2^-150);
                # the sum of exponentials is good to 2^-22 of itself
                assert abs(g - w) <= 2.0 ** -150 + 2.0 ** -24 * abs(w) + 2.0 ** -22 * min(1.0, -np.expm1(-abs(w))) + 2.0 ** -22 * abs(w), (what, i, g, w)


def logits(rows, vocab, dtype, seed=0, spread=2.0):
    rng = np.random.RandomState(seed + vocab)
    x = spread * rng.randn(rows, vocab)
    for i in range(rows):
        x[i, rng.randint(0, vocab, 4)] += 3 * spread
    return L.rounded(x, dtype), np.float32(rng.rand(rows))


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.01),
            (0.0, 7, 0.5, 0.5), (2.0, 300, 0.999, 0.0), (0.3, 1, 0.4, 0.0), (1.0, 0, 0.01, 0.0), (1.0, 0, 1.0, 1.0), (5.0, 0, 0.6, 0.001)]


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 255, 513, 1003, 2049, 4097, 8200, 20011, 40001, 70001, 140001])
def test_against_64_bits(T, vocab, dtype):
    x, u = logits(len(SETTINGS), vocab, dtype)
    got = run(T, x, u, dtype, SETTINGS, skew=vocab & 1)
    check(T, x, u, dtype, SETTINGS, got, f"{vocab} {dtype}")


@pytest.mark.parametrize("s", SETTINGS)
def test_one_descriptor_for_all_rows(T, s):
    x, u = logits(40, 3001, "bf16", 5)
    got = run(T, x, u, "bf16", temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3])
    check(T, x, u, "bf16", [s] * 40, got)


@pytest.mark.parametrize("vocab", [40, 999, 5000, 70000])
def test_ties(T, vocab):
    """Few different logits: the filters' borders lie among equal ones, of which the first by index are left."""
    rng = np.random.RandomState(vocab)
    x = rng.randint(0, 4, (24, vocab)).astype(np.float64)
    x[:6] = 1.5                                         # all equal
    x[6:8] = np.where(rng.rand(2, vocab) < 0.5, 0.0, -0.0)   # zeros of either sign are equal
    settings = [(1.0, [3, 17, 0, vocab // 2][i % 4], [1.0, 0.37, 0.71][i % 3], 0.0) for i in range(24)]
    for dtype in ("bf16", "f32"):
        u = np.float32(rng.rand(24))
        check(T, x, u, dtype, settings, run(T, x, u, dtype, settings), f"ties {vocab}")


@pytest.mark.parametrize("vocab", [10, 3000, 70000])
def test_masks_and_exceptional_rows(T, vocab):
    x, u = logits(10, vocab, "f32", 3)
    x[0, 1:] = -np.inf                     # a single token
    x[1] = -np.inf                         # none
    x[2, vocab // 2] = np.nan
    x[3, vocab // 2] = np.inf
    x[4, ::2] = -np.inf
    x[5] = np.float64(np.float32(-3.0e38))
    x[6] = np.where(np.arange(vocab) % 3 == 0, 3.0e38, -3.0e38)
    x[7] = 1e-3 * x[7]
    x[8] = 1e4 * x[8]
    x[9, 0] = -np.finfo(np.float32).max
    x = L.rounded(x, "f32")
    for s in [(1.0, 0, 1.0, 0.0), (0.9, 3, 1.0, 0.0), (1.0, 0, 0.8, 0.0), (1.1, 0, 1.0, 0.2), (0.0, 0, 1.0, 0.0), (0.8, vocab // 2, 0.9, 1e-4)]:
        check(T, x, u, "f32", [s] * 10, run(T, x, u, "f32", [s] * 10), f"{s}")


def test_random_numbers_at_the_ends(T):
    x, _ = logits(8, 1500, "f32", 9)
    u = np.array([0.0, -1.0, np.nan, 1.0, 2.0, np.inf, np.nextafter(np.float32(1), np.float32(0)), 1e-30], np.float32)
    for s in ((1.0, 0, 1.0, 0.0), (1.0, 20, 0.9, 0.0)):
        got = run(T, x, u, "f32", [s] * 8)
        for i in range(8):
            left = np.sort(np.argsort(-x[i], kind="stable")[:got[1][i]])
            assert got[0][i] == (left[-1] if u[i] > 0.5 else left[0])


def test_settings_out_of_range(T):
    x, u = logits(9, 700, "bf16", 11)
    odd = [(-1.0, 0, 1.0, 0.0), (np.nan, 0, 1.0, 0.0), (np.inf, 0, 1.0, 0.0), (1.0, -5, 1.0, 0.0), (1.0, 10 ** 6, 1.0, 0.0), (1.0, 0, 7.0, 0.0),
           (1.0, 0, np.nan, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1.0, 3.0)]
    same = [(0.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1e30, 0, 1.0, 0.0)] + [(1.0, 0, 1.0, 0.0)] * 4 + [(1.0, 1, 1.0, 0.0), (1.0, 0, 1.0, 1.0)]
    got = run(T, x, u, "bf16", odd)
    check(T, x, u, "bf16", same, got)
    got = run(T, x[:1], u[:1], "bf16", [(1.0, 0, 1.0, np.nan)])
    check(T, x[:1], u[:1], "bf16", [(1.0, 0, 1.0, 0.0)], got)


def test_one_token_has_nearly_all(T):
    """The log-probability of a token that is all but certain keeps its figures."""
    x = np.full((4, 90), -40.0)
    x[:, 7] = 0.0
    x[:, 8] = [-20.0, -12.5, -30.0, -25.0]
    s = [(1.0, 0, 1.0, 0.0), (1.0, 2, 1.0, 0.0), (0.9, 0, 1.0, 0.0), (1.2, 0, 0.99999, 0.0)]
    got = run(T, x, np.full(4, 0.25, np.float32), "f32", s)
    for i in range(4):
        token, kept, logp, logq, _ = draw(x[i], 0.25, f32(s[i][0]), s[i][1], f32(s[i][2]), 0.0)
        assert got[0][i] == token == 7
        assert abs(got[2][i] - logp) <= 2.0 ** -21 * abs(logp) and abs(got[3][i] - logq) <= 2.0 ** -21 * abs(logq)


def test_strides_and_optional_results(T):
    x, u = logits(6, 500, "f16", 13)
    wide = np.concatenate([x, np.full((6, 21), 60.0)], 1)
    want = run(T, x, u, "f16", top_p=0.9)
    got = run(T, wide, u, "f16", ld=521, vocab=500, top_p=0.9)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    tok = Buf(T, np.zeros(6, np.int32), "i32")
    T.sample_tokens(6, 500, Buf(T, x, "f16"), Buf(T, u), tok, top_p=0.9, dtype="f16")
    assert np.array_equal(tok.bits(), want[0])
    T.sample_tokens(0, 500, tok, tok, tok, dtype="f16")


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.8, top_k=30), dict(top_p=0.8)])
def test_frequencies(T, kw):
    """Over evenly spread random numbers every token comes up as often as its probability says, but for one at either end."""
    n, vocab = 4000, 50
    x, _ = logits(1, vocab, "f32", 21)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = run(T, np.repeat(x, n, 0), u, "f32", **kw)
    order = np.argsort(-x[0], kind="stable")
    w = np.zeros(vocab)
    left = order[:got[1][0]]
    w[left] = np.exp((x[0, left] - x.max()) / f32(kw.get("temperature", 1.0)))
    counts = np.bincount(got[0], minlength=vocab)
    assert (np.abs(counts - n * w / w.sum()) <= 1.001).all()
    assert (np.diff(got[0]) >= 0).all()


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.9])
@pytest.mark.parametrize("rows,vocab", [(5, 9001), (600, 8200), (9, 70001), (3, 200003)])
def test_long_rows_without_filters(T, rows, vocab, temperature, dtype):
    """One descriptor that leaves all, few rows and more than twice the compute units."""
    x, u = logits(rows, vocab, dtype, 4)
    got = run(T, x, u, dtype, temperature=temperature)
    some = np.unique(np.concatenate([np.arange(min(rows, 12)), [rows - 1]]))
    check(T, x[some], u[some], dtype, [(temperature, 0, 1.0, 0.0)] * len(some), [g[some] for g in got], f"{rows} x {vocab} {dtype}")


@pytest.mark.parametrize("vocab", [9001, 70001])
def test_masks_and_exceptional_long_rows_without_filters(T, vocab):
    x, u = logits(22, vocab, "f32", 3)
    x[0, 1:] = -np.inf                     # a single token, at the start, at the end and in between
    x[1, :-1] = -np.inf
    x[2] = -np.inf
    x[2, vocab // 2 + 333] = -77.0
    x[3] = -np.inf                         # none
    x[4, vocab // 2], x[5, vocab - 1] = np.nan, np.inf
    x[6, ::2] = -np.inf
    x[7] = -3.0e38
    x[8] = np.where(np.arange(vocab) % 3 == 0, 3.0e38, -3.0e38)
    x[9], x[10] = 1e-3 * x[9], 1e4 * x[10]
    x[11, 0] = -np.finfo(np.float32).max
    for i, shift in ((12, -50.0), (13, -1e5), (14, 50.0), (15, 1e5)):   # little is left, far from zero
        keep = np.arange(vocab) >= vocab - 5
        x[i] = np.where(keep, x[i] + shift, -np.inf)
    x[16, vocab // 3] += 70.0              # the maximum far above the others, all but certain, and the first
    x[17, vocab - 2] += 9.0 + np.log(vocab)
    x[18, 0] += 300.0
    x[19] -= 1e5
    x[20, :vocab - vocab // 50] = -np.inf
    x[20] -= 60.0
    x[21] = 0.0
    x = L.rounded(x, "f32")
    for t in (1.0, 0.9, 0.01, 30.0):
        check(T, x, u, "f32", [(t, 0, 1.0, 0.0)] * len(u), run(T, x, u, "f32", temperature=t), f"{t}")


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("rows", [1, 11, 64, 65])
@pytest.mark.parametrize("s", [(1.0, 0, 0.9, 0.0), (0.8, 0, 0.99, 0.001), (1.5, 0, 0.3, 0.0)])
def test_long_rows_with_top_p(T, rows, dtype, s):
    """Rows that several workgroups look at, and one more of them than have that."""
    vocab = 66001
    x, u = logits(rows, vocab, dtype, 6)
    x[0, : vocab // 2] = -np.inf
    got = run(T, x, u, dtype, temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3])
    some = np.unique(np.concatenate([np.arange(min(rows, 8)), [rows - 1]]))
    check(T, x[some], u[some], dtype, [s] * len(some), [g[some] for g in got], f"{rows} {dtype}")
    tok = Buf(T, np.zeros(rows, np.int32), "i32")
    T.sample_tokens(rows, vocab, Buf(T, x, dtype), Buf(T, u), tok, temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3], dtype=dtype)
    assert np.array_equal(tok.bits(), got[0])


@pytest.mark.parametrize("vocab", [66001, 140001])
@pytest.mark.parametrize("s", [(1.0, 0, 0.8, 0.0), (0.9, 0, 0.95, 1e-4), (30.0, 0, 0.5, 0.0), (0.01, 0, 0.999, 0.0)])
def test_masks_and_exceptional_long_rows_with_top_p(T, vocab, s):
    x, u = logits(16, vocab, "f32", 3)
    x[0, 1:], x[1, :-1], x[2] = -np.inf, -np.inf, -np.inf
    x[3, vocab // 2], x[4, vocab - 1], x[5, 0] = np.nan, np.inf, np.nan
    x[6, ::2] = -np.inf
    x[7] = -3.0e38
    x[8] = np.where(np.arange(vocab) % 3 == 0, 3.0e38, -3.0e38)
    x[9], x[10] = 1e-3 * x[9], 1e4 * x[10]
    x[11] = np.round(x[11])
    x[12] = np.where(np.arange(vocab) >= vocab - 5, x[12] - 50, -np.inf)
    x[13, vocab // 3] += 70.0
    x[14] = 0.0
    x[15, : vocab // 2] = -np.finfo(np.float32).max
    x = L.rounded(x, "f32")
    check(T, x, u, "f32", [s] * 16, run(T, x, u, "f32", temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3]), f"{s}")
    check(T, x, u, "f32", [s] * 16, run(T, x, u, "f32", [s] * 16), f"own {s}")
