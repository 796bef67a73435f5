"""What the tests of the language-model operators share: 16-bit types in numpy, the operators in 64 bits, and how
far a kernel may be from them."""
import numpy as np

DTYPES = ["f32", "bf16", "f16"]
HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # of a rounding, relative to the value
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}           # the smallest step of the type
NP = {"f32": np.float32, "bf16": np.uint16, "f16": np.uint16}


def encode(a, dtype):
    """float values as the bits of the type (to nearest, ties to even)."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == "f32":
        return a
    if dtype == "f16":
        return a.astype(np.float16).view(np.uint16)
    u = a.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def decode(a, dtype):
    """The bits of the type as float64."""
    if dtype == "f32":
        return a.astype(np.float64)
    if dtype == "f16":
        return a.view(np.float16).astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(a, dtype):
    return decode(encode(a, dtype), dtype)


def within(got, want, bound, what=""):
    """|got - want| <= bound element by element; what is not finite has to be the same."""
    got, want, bound = (np.asarray(v, np.float64) for v in (got, want, bound))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    off = np.abs(np.where(fine, got, 0) - np.where(fine, want, 0))
    bad = fine & ~(off <= np.broadcast_to(bound, want.shape))
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, off, 0)), want.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {want.size} too far off; at {i} got {got[i]!r}, want {want[i]!r}, "
                             f"bound {np.broadcast_to(bound, want.shape)[i]:.3g}")


# ------------------------------------------------------------------ dropout

def philox_words(n, seed, offset):
    """Philox4x32-10: word i % 4 of counter (i // 4, offset), key seed."""
    m32 = (1 << 32) - 1
    c = [np.arange((n + 3) // 4, dtype=np.uint64) & np.uint64(m32), np.arange((n + 3) // 4, dtype=np.uint64) >> np.uint64(32),
         np.full((n + 3) // 4, offset & m32, np.uint64), np.full((n + 3) // 4, offset >> 32, np.uint64)]
    k0, k1 = seed & m32, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & np.uint64(m32), (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1),
             a & np.uint64(m32)]
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return np.stack(c, 1).reshape(-1)[:n].astype(np.uint32)


def kept(n, rate, seed, offset):
    return philox_words(n, seed, offset) >= np.uint32(int(np.float64(np.float32(rate)) * 2.0 ** 32))


# ------------------------------------------------------- gated feed-forward

def gate(kind, g):
    """The activation and its derivative."""
    from scipy.special import erfc, expit
    if kind == "silu":
        s = expit(g)
        return g * s, s + g * s * (1 - s)
    if kind == "sigmoid":
        s = expit(g)
        return s, s * (1 - s)
    if kind == "gelu":
        cdf = 0.5 * erfc(-g / np.sqrt(2))
        return g * cdf, cdf + g * np.exp(-g * g / 2) / np.sqrt(2 * np.pi)
    if kind == "gelu_tanh":
        k = np.sqrt(2 / np.pi)
        t = np.tanh(k * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    if kind == "relu":
        return np.maximum(g, 0), (g > 0).astype(np.float64)
    return g, np.ones_like(g)


def ff_forward(x, w, b, act):
    z = x @ w + (0 if b is None else b)
    g, u = np.split(z, 2, 1)
    return z, gate(act, g)[0] * u


def ff_backward(x, w, z, dh, act):
    g, u = np.split(z, 2, 1)
    a, da = gate(act, g)
    dz = np.concatenate([dh * u * da, dh * a], 1)
    return dz, dz @ w.T, x.T @ dz, dz.sum(0)


def sum_bound(terms, magnitude):
    """An fp32 sum of products of `terms` terms whose absolute values add up to `magnitude`: at most two roundings
    (or truncations, 2^-23 each) a term, and a few more where partial sums meet."""
    return (2 * terms + 16) * 2.0 ** -23 * magnitude


ACT_SLOPE = 1.2    # no gate's derivative is larger (gelu's 1.13)
ACT_CURVE = 1.0    # nor its second derivative (gelu's 0.8)
ACT_REL = 2.0 ** -18   # of an activation or derivative in fp32, of its terms (|g| of 20 in an exponent: 20 roundings)


def ff_forward_bounds(x, w, b, act, dtype):
    z, h = ff_forward(x, w, b, act)
    g, u = np.split(z, 2, 1)
    dz = sum_bound(x.shape[1], np.abs(x) @ np.abs(w) + (0 if b is None else np.abs(b)))
    dg, du = np.split(dz, 2, 1)
    a = np.abs(gate(act, g)[0])
    dh = ACT_SLOPE * dg * (np.abs(u) + du) + a * du + ACT_REL * (np.abs(g) + 1) * np.abs(u)
    dh = dh + HALF_ULP[dtype] * (np.abs(h) + dh) + TINY[dtype]
    return (z, dz + 2.0 ** -24 * np.abs(z)), (h, dh)


def ff_backward_bounds(x, w, z, dh, act, dtype):
    """z: as the kernel reads it."""
    dz, dx, dw, db = ff_backward(x, w, z, dh, act)
    g, u = np.split(z, 2, 1)
    off = np.abs(np.concatenate([dh * u, dh * (np.abs(g) + 1)], 1)) * ACT_REL * (1 + np.abs(np.concatenate([g, g], 1))) + 2.0 ** -22 * np.abs(dz)
    half = off + (HALF_ULP[dtype] * (np.abs(dz) + off) + TINY[dtype] if dtype != "f32" else 0)  # (rounded as an operand)

    def final(v, e):
        return e + HALF_ULP[dtype] * (np.abs(v) + e) + TINY[dtype]

    n, m = dz.shape
    return {"dx": (dx, final(dx, half @ np.abs(w).T + sum_bound(m, (np.abs(dz) + half) @ np.abs(w).T))),
            "dw": (dw, final(dw, np.abs(x).T @ half + sum_bound(n, np.abs(x).T @ (np.abs(dz) + half)))),
            "db": (db, final(db, half.sum(0) + sum_bound(n, (np.abs(dz) + half).sum(0))))}


# ------------------------------------------------------------------- losses

def logprob(x, target):
    """(logp, (m, s), p, counted) of rows of float64 logits; a target past the end gives NaN."""
    with np.errstate(all="ignore"):
        live = target >= 0
        m = np.max(x, 1, initial=-np.inf)
        m0 = np.where(np.isfinite(m), m, np.where(m > 0, m, 0.0))
        e = np.exp(x - m0[:, None])
        total = e.sum(1)
        t = np.where((target >= 0) & (target < x.shape[1]), target, 0)
        logp = np.where(target >= x.shape[1], np.nan, x[np.arange(len(x)), t] - m0 - np.log(total))
        p = e / total[:, None]
    return np.where(live, logp, 0.0), np.where(live[:, None], np.stack([m0, total], 1), 0.0), p, live


def dlogits(x, target, d):
    _, _, p, live = logprob(x, target)
    with np.errstate(all="ignore"):
        g = -p * d[:, None]
        for r in np.flatnonzero(live):
            if target[r] < x.shape[1]:
                g[r, target[r]] += d[r]
            else:
                g[r] = np.nan
    return np.where(live[:, None], g, 0.0)


def policy(logp, target, old, ref, adv, weight, low, high, kl):
    """(row losses, factors of the gradient)"""
    with np.errstate(all="ignore"):
        w = np.ones_like(logp) if weight is None else weight
        r = np.exp(logp - old)
        free, held = r * adv, np.clip(r, 1 - low, 1 + high) * adv
        loss, d = -np.minimum(free, held), np.where(free <= held, -free, np.where(free > held, 0.0, np.nan))
        if ref is not None:
            gap = ref - logp
            loss, d = loss + kl * (np.expm1(gap) - gap), d - kl * np.expm1(gap)
        live = target >= 0
        return np.where(live, w * loss, 0.0), np.where(live, w * d, 0.0)


def preference(seq, ref, beta, smoothing, kind):
    """(margins, losses of the pairs, factors of the gradient of the mean loss by sequence)"""
    ratio = seq - (0 if ref is None else ref)
    m = beta * (ratio[0::2] - ratio[1::2])
    if kind == "sigmoid":
        loss = (1 - smoothing) * np.logaddexp(0, -m) + smoothing * np.logaddexp(0, m)
        from scipy.special import expit
        dm = smoothing * expit(m) - (1 - smoothing) * expit(-m)
    elif kind == "squared":
        loss, dm = ((m - 0.5) / beta) ** 2, 2 * (m - 0.5) / beta ** 2
    else:
        loss, dm = np.maximum(0, 1 - m), -(m < 1).astype(np.float64)
    d = beta * dm / len(m)
    return m, loss, np.stack([d, -d], 1).reshape(-1)


def lse_bound(x):
    """The log-sum's error: what its terms' exponents round off (their distance from the maximum, weighted by what
    they are worth), a thread's fp32 sum of at most 128 terms, and the rounding of the result."""
    v = x.shape[1]
    return 2.0 ** -23 * (np.log(v) + 8) + 128 * 2.0 ** -24


def dlogits_bound(x, target, d, d_off, dtype):
    """d_off: the error of d."""
    _, _, p, live = logprob(x, target)
    with np.errstate(all="ignore"):
        far = np.abs(x - np.max(x, 1)[:, None])
        far = np.where(np.isfinite(far), far, 0)
        rel = 2.0 ** -22 * (far + 4) + lse_bound(x)
        hit = np.zeros_like(x)
        ok = live & (target < x.shape[1])
        hit[np.flatnonzero(ok), target[ok]] = 1.0
        want = np.abs(dlogits(x, target, d))
        off = p * np.abs(d)[:, None] * rel + (p + hit) * np.asarray(d_off)[:, None] + 2.0 ** -23 * np.abs(d)[:, None] * hit
        off = off + HALF_ULP[dtype] * (want + off) + TINY[dtype] + 2.0 ** -126 * np.abs(d)[:, None]  # (exponents below 2^-126 may be flushed)
    return np.where(np.isfinite(off), off, 0) * live[:, None]
