"""The operators of learning from a model's own answers, in the order of a turn: a normalised layer's logits in 8 bits, tokens drawn from them, the
policy loss of those tokens under the full logits, the way back through the normalisation, and the matrix's update. Against the same in 64 bits."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import lm_common as L  # noqa: E402
import test_gpu_layernorm as N  # noqa: E402
import test_gpu_muon as M  # noqa: E402
import test_gpu_sample_tokens as S  # noqa: E402
from test_gpu_fc_q8 import Bytes, quantized  # noqa: E402
from test_gpu_lm_operators import Buf, out  # noqa: E402

pytestmark = pytest.mark.gpu

# a product's factors and the sums of up to 64 of them: 64 additions and a few roundings of each factor, 2^-24 each, along three products in a row
SUM = 2.0 ** -16


@pytest.mark.parametrize("dtype", L.DTYPES)
def test_turns(T, dtype):
    n, d, v = 48, 64, 61
    rng = np.random.RandomState(3)
    x, gamma, beta = (L.rounded(a, dtype) for a in (rng.randn(n, d), 1 + 0.1 * rng.randn(d), 0.1 * rng.randn(d)))
    w, mom = L.rounded(rng.randn(d, v) / 8, "f32"), np.zeros((d, v))
    bw, bmom = Buf(T, w), Buf(T, mom)
    bx, bgamma, bbeta = (Buf(T, a, dtype) for a in (x, gamma, beta))
    opt = T.muon_desc(alpha=0.05)
    kw = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.001)
    for turn in range(3):
        u = np.float32(rng.rand(n))
        adv = L.rounded(rng.randn(n), "f32")
        # the answers
        wq, ws = Bytes(T, np.full((v, T.q8_row(d)), 3, np.int8)), out(T, v)
        y, stats, rough = out(T, (n, d), dtype), out(T, (n, 2)), out(T, (n, v))
        token, old = Buf(T, np.full(n, -7, np.int32), "i32"), out(T, n)
        T.fc_q8_pack(d, v, bw, wq, ws)
        T.layernorm_fwd(n, d, bx, bgamma, bbeta, y, stats, dtype=dtype)
        yf = y
        if dtype != "f32":
            yf = out(T, (n, d))
            T.cast(n * d, y, yf, dtype, "f32")
        T.fc_q8_fwd(d, v, False, n, yf, wq, ws, None, rough)
        T.sample_tokens(n, v, rough, Buf(T, u), token, old, **kw)
        # the gradient
        logits, logp, total, dl = out(T, (n, v)), out(T, n), out(T, 1), out(T, (n, v))
        dy, dw, dx, dgamma, dbeta = out(T, (n, d)), out(T, (d, v)), out(T, (n, d), dtype), out(T, d, dtype), out(T, d, dtype)
        T.fc_fwd(d, v, False, n, yf, bw, None, logits)
        T.policy_loss(n, v, logits, token, old, None, Buf(T, adv), None, logp, None, total, dl)
        T.fc_bwd(d, v, False, n, yf, bw, dl, dy, dw, None)
        dyt = dy
        if dtype != "f32":
            dyt = out(T, (n, d), dtype)
            T.cast(n * d, dy, dyt, "f32", dtype)
        T.layernorm_bwd(n, d, bx, bgamma, stats, dyt, dx, dgamma, dbeta, dtype=dtype)
        # and the update
        T.muon_update(opt, d, v, dw, bw, bmom)

        # the same in 64 bits, each link from what the one before gave where that was rounded to the type
        t = N.truth(x, gamma, beta, dyt.read())
        near = N.bounds(x, t, gamma, beta, dyt.read(), dtype, n)
        for got, k in ((y, "y"), (dx, "dx"), (dgamma, "dgamma"), (dbeta, "dbeta")):
            L.within(got.read(), t[k], near[k], f"{k} of turn {turn}")
        h = y.read()
        qx, sx = quantized(h)
        qw, sw = quantized(w.T)
        assert np.array_equal(wq.read()[:, :d], qw) and np.array_equal(ws.read(), sw)
        want = (qx @ qw.T) * sx[:, None] * sw
        L.within(rough.read(), want, 4 * 2.0 ** -24 * np.abs(want), "8-bit logits")
        drawn = 0
        for i in range(n):
            one, _, lp, _, margin = S.draw(rough.read()[i], u[i], S.f32(0.8), 40, S.f32(0.95), S.f32(0.001))
            if margin > 1e-9:
                drawn += 1
                assert token.bits()[i] == one, (turn, i)
                assert abs(old.read()[i] - lp) <= 2.0 ** -21 * max(1.0, abs(lp))
        assert drawn >= n - 1
        tok, was = token.bits(), old.read()

        def loss_of(h, w):
            return L.policy(L.logprob(h @ w, tok)[0], tok, was, None, adv, None, 0.2, 0.2, 0.0)[0].sum()

        size = np.abs(h) @ np.abs(w)                                # of the logits' sums
        now = L.logprob(h @ w, tok)[0]
        L.within(logp.read(), now, SUM * (1 + size.max(1) + np.abs(now)), "log-probabilities")
        assert np.abs(np.abs(np.exp(now - was) - 1) - 0.2).min() > 1e-3     # no row on the border of the clip
        L.within(total.read(), [loss_of(h, w)], SUM * (np.abs(adv) * (2 + size.max(1))).sum(), "loss")
        g = L.dlogits(h @ w, tok, L.policy(now, tok, was, None, adv, None, 0.2, 0.2, 0.0)[1])
        eg = SUM * (np.abs(adv) * (2 + size.max(1)))[:, None]        # a gradient's entry is below 1.2 times the advantage
        L.within(dl.read(), g, eg, "gradient of the logits")
        L.within(dy.read(), g @ w.T, eg * np.abs(w).sum(1) + SUM * np.abs(g) @ np.abs(w.T), "dy")
        L.within(dw.read(), h.T @ g, np.abs(h.T) @ np.broadcast_to(eg, g.shape) + SUM * np.abs(h.T) @ np.abs(g), "dw")
        for i in ((0, 0), (17, 30), (63, 60)):                       # the chain in 64 bits against differences
            e = np.zeros_like(w)
            e[i] = 1e-6
            assert abs((loss_of(h, w + e) - loss_of(h, w - e)) / 2e-6 - (h.T @ g)[i]) < 1e-5 * (1 + abs((h.T @ g)[i]))
        grad = dw.read()
        mom = M.f32(0.95) * mom + grad
        L.within(bmom.read(), mom, 3 * 2.0 ** -24 * (np.abs(mom) + np.abs(grad)), "momentum")
        o = M.start(grad + M.f32(0.95) * mom)
        e, flat = 40 * M.U * np.linalg.norm(o), 1.0 / v
        for _ in range(5):
            e = 4 * e + np.linalg.norm(M.step_bound(o, "f32", flat))
            o, s = M.step(o), np.sqrt(flat)
            flat = (s * (M.a + M.b * flat + M.c * flat * flat)) ** 2
        want = w - M.f32(0.05) * o
        assert np.linalg.norm(bw.read() - want) <= M.f32(0.05) * e + 8 * M.U * np.linalg.norm(w)
        w, mom = bw.read(), bmom.read()


@pytest.mark.parametrize("dtype", L.DTYPES)
@pytest.mark.parametrize("vocab", [61, 5003, 70001])
def test_the_ratio_of_a_first_step_is_one(T, dtype, vocab):
    """Drawn from the very logits that learn, a token's old log-probability is its new one: the loss is the advantages' sum taken off, whatever was cut
    off before the draw, and a masked token is neither drawn nor weighed."""
    rows = 9
    x, u = S.logits(rows, vocab, dtype, 1)
    x[:, ::7] = -np.inf
    rng = np.random.RandomState(vocab)
    adv = L.rounded(rng.randn(rows), "f32")
    bx, token, old, logp, each, total = Buf(T, x, dtype), Buf(T, np.full(rows, -7, np.int32), "i32"), out(T, rows), out(T, rows), out(T, rows), out(T, 1)
    T.sample_tokens(rows, vocab, bx, Buf(T, u), token, old, temperature=0.7, top_k=50, top_p=0.9, dtype=dtype)
    T.policy_loss(rows, vocab, bx, token, old, None, Buf(T, adv), None, logp, each, total, None, dtype=dtype)
    assert (token.bits() % 7 != 0).all() and (token.bits() >= 0).all()
    # either log-probability: a rounding of the result and of the logarithm, 2^-22 of the sum, and of the distance to the maximum in the exponent
    off = 2.0 ** -20 * (1 + np.abs(old.read()))
    L.within(logp.read(), old.read(), off, "log-probabilities")
    L.within(each.read(), -adv, np.abs(adv) * (2 * off + 2.0 ** -22), "losses")
    L.within(total.read(), [-adv.sum()], (np.abs(adv) * (2 * off + 2.0 ** -20)).sum(), "loss")
