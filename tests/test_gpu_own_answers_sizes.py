"""Layer normalisation, drawn tokens, 8-bit products and the orthogonalised update at the ends of their ranges: rows whose offsets pass 32 bits, many rows, the longest sides."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
import test_gpu_fc_q8 as Q  # noqa: E402
import test_gpu_layernorm as N  # noqa: E402
import test_gpu_muon as M  # noqa: E402
import test_gpu_sample_tokens as S  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu


class FarRows:
    """Rows of fp32 numbers `ld` elements apart, with nothing in between."""

    def __init__(self, T, values, ld):
        self.T, self.shape, self.ld = T, values.shape, ld
        self.buf = T.DevBuf(4 * ((len(values) - 1) * ld + values.shape[1]), np.uint8)
        self.ptr = self.buf.ptr
        for i, v in enumerate(values):
            self.row(i).upload(v)

    def row(self, i):
        return self.T.DevBuf.view(self.buf.ptr.value + 4 * i * self.ld, self.shape[1:], np.float32)

    def read(self):
        return np.stack([self.row(i).numpy() for i in range(self.shape[0])]).astype(np.float64)


LD = 1_200_000_001   # the third row begins 9.6 GB behind the first one, its elements past 2^31


@pytest.mark.parametrize("n", [300, 9001])
def test_layernorm_of_rows_far_apart(T, n):
    x, gamma, beta, dy = N.case(3, n, "f32")
    t = N.truth(x, gamma, beta, dy)
    b = N.bounds(x, t, gamma, beta, dy, "f32", 3)
    bx, bdy, by = FarRows(T, x, LD), FarRows(T, dy, LD), FarRows(T, 0 * x, LD)
    bg, bb, st, dg, db = Buf(T, gamma), Buf(T, beta), out(T, (3, 2)), out(T, n), out(T, n)
    T.layernorm_fwd(3, n, bx, bg, bb, by, st, ld=LD, ld_y=LD)
    L.within(by.read(), t["y"], b["y"], "y")
    T.layernorm_bwd(3, n, bx, bg, st, bdy, by, dg, db, ld=LD, ld_dy=LD, ld_dx=LD)
    for got, k in ((by, "dx"), (dg, "dgamma"), (db, "dbeta")):
        L.within(got.read(), t[k], b[k], k)


@pytest.mark.parametrize("vocab", [300, 5003, 70001])
def test_tokens_of_rows_far_apart(T, vocab):
    x, u = S.logits(3, vocab, "f32", 2)
    bx, bu = FarRows(T, x, LD), Buf(T, u)
    for s in ((1.0, 0, 1.0, 0.0), (0.9, 0, 0.9, 0.0), (1.0, 30, 0.95, 0.01)):
        tok, kept, logp, logq = out(T, 3), out(T, 3), out(T, 3), out(T, 3)
        tok.dtype = kept.dtype = "i32"
        T.sample_tokens(3, vocab, bx, bu, tok, logp, logq, kept, temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3], ld=LD)
        S.check(T, x, u, "f32", [s] * 3, (tok.bits(), kept.bits(), logp.read(), logq.read()), f"{vocab} {s}")


def test_many_rows(T):
    n, d = 200001, 24
    x, gamma, beta, dy = N.case(n, d, "f16")
    t = N.truth(x, gamma, beta, dy)
    b = N.bounds(x, t, gamma, beta, dy, "f16", n)
    got = N.run(T, x, gamma, beta, dy, "f16")
    for k in b:
        L.within(got[k], t[k], b[k], k)
    rng = np.random.RandomState(3)
    n, d, f = 70001, 40, 24
    x = L.rounded(rng.randn(n, d), "bf16")
    wq, ws = Q.weights(rng, d, f)
    y = out(T, (n, f), "bf16")
    T.fc_q8_fwd(d, f, False, n, Buf(T, x, "bf16"), Q.Bytes(T, wq), Buf(T, ws), None, y, dtype="bf16")
    want, _ = Q.truth(x, wq, ws, None)
    L.within(y.read(), want, Q.bound(want, np.zeros(1), "bf16"), "q8")
    rows, vocab = 80000, 17
    x, u = L.rounded(2 * rng.randn(rows, vocab), "f16"), np.float32(rng.rand(rows))
    got = S.run(T, x, u, "f16", temperature=0.8, top_k=6, top_p=0.9)
    some = np.concatenate([np.arange(40), np.arange(rows - 40, rows)])
    S.check(T, x[some], u[some], "f16", [(0.8, 6, 0.9, 0.0)] * len(some), [g[some] for g in got])


@pytest.mark.parametrize("shape", [(3, 1 << 20), (1 << 20, 3)])
@pytest.mark.parametrize("products", ["f32", "f16"])
def test_the_longest_side_of_an_update(T, shape, products):
    u = M.matrix(*shape, "f32")
    y = out(T, shape)
    T.orthogonalize(T.muon_desc(steps=1, products=products), *shape, Buf(T, u), y)
    x = M.start(u)
    want, e = M.step(x), M.step_bound(x, products, 1.0 / 3) + 12 * M.U * np.abs(x)
    L.within(y.read(), want, e + 5 * M.U * np.abs(want), f"{shape} {products}")
