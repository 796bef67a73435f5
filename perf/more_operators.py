"""More operators of language models as cases that can be timed, what training a model by its own answers takes beside the losses:
products in 8-bit integers and the drawing of tokens, with which answers are written, and layer normalisation with its gradients
and the orthogonalised update, with which the model learns from them.

A case is a dict of plain values; ``listed()`` names the ones that are followed, ``draw(rng)`` gives others of the same
ranges. ``run`` computes an operator in elementary torch operations, or, where ``own`` is true, by the calls of this library
on the same buffers. ``exact`` says what the definitions give in 64 bits.
"""
import ctypes
import importlib
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # Behind a small net's hidden layer (batch 37, 64 units), forward and backward: the time of the launches.
        {"name": "norm_small_f32", "op": "norm", "dtype": "f32", "rows": 37, "len": 64},
        # Ragged: neither the rows nor their length are a multiple of anything.
        {"name": "norm_odd_f16", "op": "norm", "dtype": "f16", "rows": 501, "len": 1001},
        # A training step's tokens through one normalisation of a large model, there and back.
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bf16", "rows": 8192, "len": 4096},
        # The update of a small net's fully-connected layer.
        {"name": "muon_small_f32", "op": "muon", "dtype": "f32", "rows": 120, "cols": 84, "steps": 5},
        # The update of the fully-connected benchmark's weights, in fp32 throughout.
        {"name": "muon_f32", "op": "muon", "dtype": "f32", "rows": 4096, "cols": 4096, "steps": 5},
        # A large model's gradient in 16 bits, of a gated block's gate or up weights.
        {"name": "ortho_bf16", "op": "ortho", "dtype": "bf16", "rows": 4096, "cols": 12288, "steps": 5},
        # One answer being written: a row, everything switched on.
        {"name": "sample_one_f32", "op": "sample", "dtype": "f32", "rows": 1, "vocab": 50003, "temperature": 0.8, "top_k": 50,
         "top_p": 0.95, "min_p": 0.01, "per_row": False, "masked": 0.0},
        # A server's batch, each of its rows with settings of its own, half of them under a grammar's mask.
        {"name": "sample_batch_bf16", "op": "sample", "dtype": "bf16", "rows": 64, "vocab": 131072, "temperature": 0.9, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "per_row": True, "masked": 0.5},
        # Answers for training: the model's own distribution, as it is.
        {"name": "sample_rollout_bf16", "op": "sample", "dtype": "bf16", "rows": 2048, "vocab": 65536, "temperature": 1.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "per_row": False, "masked": 0.0},
        # One token through a layer whose weights are held in 8 bits.
        {"name": "q8_token_bf16", "op": "q8", "dtype": "bf16", "n_in": 4096, "n_out": 12288, "batch": 1, "bias": False},
        # A ragged handful of rows where no size is a multiple of anything.
        {"name": "q8_odd_f16", "op": "q8", "dtype": "f16", "n_in": 1001, "n_out": 2731, "batch": 77, "bias": True},
        # A long prompt.
        {"name": "q8_prompt_bf16", "op": "q8", "dtype": "bf16", "n_in": 4096, "n_out": 12288, "batch": 4096, "bias": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["norm", "norm", "muon", "ortho", "sample", "sample", "q8", "q8"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "norm":
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 20_000), "len": _log_int(rng, 2, 20_000)}
    if op in ("muon", "ortho"):
        round_to = rng.choice([1, 1, 8, 64])
        rows, cols = (max(round_to, _log_int(rng, 4, 4000) // round_to * round_to) for _ in range(2))
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "steps": rng.choice([4, 5, 5, 6])}
    if op == "sample":
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 3000), "vocab": _log_int(rng, 2, 140_000),
                "temperature": round(rng.uniform(0.3, 1.5), 3), "top_k": rng.choice([0, 0, _log_int(rng, 1, 2000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.999), 4)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]), "per_row": rng.random() < 0.5,
                "masked": rng.choice([0.0, 0.5])}
    round_to = rng.choice([1, 1, 16, 128])
    n_in, n_out = (max(round_to, _log_int(rng, 24, 8000) // round_to * round_to) for _ in range(2))
    return {"op": op, "dtype": dtype, "n_in": n_in, "n_out": n_out, "bias": rng.random() < 0.5,
            "batch": rng.choice([1, 1, _log_int(rng, 2, 4096), _log_int(rng, 2, 4096)])}


def draw(rng):
    while True:
        c = _draw_once(rng)
        w = work(c)
        if w["bytes"] <= 2.6e8 and w["flops"] <= 4.1e11:
            return c


# ------------------------------------------------------------------------ what it needs

def work(c):
    s = SIZE[c["dtype"]]
    if c["op"] == "norm":  # x, dy -> y, dx; the gains and their gradients, the rows' statistics
        return {"bytes": float(s * (4 * c["rows"] * c["len"] + 4 * c["len"]) + 8 * c["rows"]), "flops": 0.0}
    if c["op"] in ("muon", "ortho"):
        n, (m, k) = float(c["rows"]) * c["cols"], sorted((c["rows"], c["cols"]))
        moved = 2 * s if c["op"] == "ortho" else s + 16  # g -> y; or g, and the weights and the momentum in and out
        # two of the three products of a step are symmetric, and half of them is the other half
        return {"bytes": moved * n, "flops": c["steps"] * (3.0 * m * m * k + 1.0 * m * m * m)}
    if c["op"] == "sample":
        return {"bytes": float(s) * c["rows"] * c["vocab"] + 36.0 * c["rows"], "flops": 0.0}
    x, w, y = c["batch"] * c["n_in"], c["n_in"] * c["n_out"], c["batch"] * c["n_out"]
    return {"bytes": float(s * (x + y) + w + c["n_out"] * (4 + (s if c["bias"] else 0))), "flops": 2.0 * c["batch"] * w}


# ---------------------------------------------------------------------------- prepare

class _Buf:
    """A tensor's device address as the library's calls take it."""

    def __init__(self, t):
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr())


EPS = 1e-5                                    # of the normalisation
A, B, C, TINY = 3.4445, -4.7750, 2.0315, 1e-7   # the iteration's polynomial a x + b x^3 + c x^5, and what is added to the norm
ALPHA, MU, DECAY = 0.02, 0.95, 0.01


def _padded(n):
    return (n + 15) // 16 * 16


def _gradient(rows, cols, gen):
    """A weight gradient: some strong directions of falling strength, and noise."""
    k = min(32, rows, cols)
    u = torch.randn(rows, k, generator=gen, device="cuda") * torch.logspace(0, -2, k, device="cuda")
    v = torch.randn(k, cols, generator=gen, device="cuda")
    return (3.0 * (u @ v) + 0.5 * torch.randn(rows, cols, generator=gen, device="cuda")) * 1e-3


def prepare(case, seed):
    c = dict(case)
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[c["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=dev) * std

    b = {}
    if c["op"] == "norm":
        n, d = c["rows"], c["len"]
        b["x"] = (normal(n, d, std=1.5) * (1 + 4 * (torch.rand(d, generator=gen, device=dev) < 0.01)) + normal(n, 1)).to(dtype)
        b["gamma"], b["beta"] = (1 + normal(d, std=0.2)).to(dtype), normal(d, std=0.2).to(dtype)
        b["dy"] = normal(n, d).to(dtype)
        b["y"], b["dx"] = torch.zeros_like(b["x"]), torch.zeros_like(b["x"])
        b["stats"] = torch.zeros(n, 2, device=dev)
        b["dgamma"], b["dbeta"] = torch.zeros_like(b["gamma"]), torch.zeros_like(b["beta"])
    elif c["op"] in ("muon", "ortho"):
        b["g"] = _gradient(c["rows"], c["cols"], gen).to(dtype)
        if c["op"] == "ortho":
            b["y"] = torch.zeros_like(b["g"])
        else:
            b["w"] = normal(c["rows"], c["cols"], std=1.0 / math.sqrt(c["rows"]))
            b["momentum"] = 5.0 * _gradient(c["rows"], c["cols"], gen)
    elif c["op"] == "sample":
        n, v = c["rows"], c["vocab"]
        x = normal(n, v, std=2.0)
        top = torch.randint(0, v, (n, 8), generator=gen, device=dev)
        x.scatter_add_(1, top, 5.0 + normal(n, 8, std=2.0))  # what the model has in mind
        if c["masked"] > 0:
            out = torch.rand(n, v, generator=gen, device=dev) < c["masked"]
            out &= torch.rand(n, 1, generator=gen, device=dev) < 0.5  # of half of the rows
            x.masked_fill_(out.scatter_(1, top[:, :1], False), -math.inf)
        b["logits"] = x.to(dtype)
        b["u"] = torch.rand(n, generator=gen, device=dev)
        if c["per_row"]:  # around the case's settings: temperature, top_k, top_p, min_p
            r = torch.rand(4, n, generator=gen, device=dev)
            t = (c["temperature"] * (0.8 + 0.4 * r[0])).float()
            k = (c["top_k"] * (0.5 + r[1])).to(torch.int32)
            p = (c["top_p"] + (1 - c["top_p"]) * (r[2] - 0.5)).float()
            q = (c["min_p"] * (0.5 + r[3])).float()
            b["settings"] = torch.stack((t.view(torch.int32), k, p.view(torch.int32), q.view(torch.int32)), 1).contiguous()
        b["token"] = torch.zeros(n, device=dev, dtype=torch.int32)
        b["kept"] = torch.zeros(n, device=dev, dtype=torch.int32)
        b["logp"], b["logq"] = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    else:
        n, d, f = c["batch"], c["n_in"], c["n_out"]
        outliers = 1 + 9 * (torch.rand(d, generator=gen, device=dev) < 0.002)
        b["x"] = (normal(n, d) * outliers).to(dtype)
        w = normal(f, d, std=1.0 / math.sqrt(d))
        b["wscale"] = w.abs().amax(1) / 127.0
        b["wq"] = torch.zeros(f, _padded(d), device=dev, dtype=torch.int8)  # an output's weights along, rows of whole words
        b["wq"][:, :d] = (w / b["wscale"][:, None]).round().to(torch.int8)
        b["b"] = normal(f, std=0.1).to(dtype) if c["bias"] else None
        b["y"] = torch.zeros(n, f, device=dev, dtype=dtype)
    return {"case": c, "t": b, "buf": {k: _Buf(t) for k, t in b.items() if t is not None}}


# ------------------------------------------------------------------------- plain forms

def _plain_norm(t):
    x, dy, dtype = t["x"].float(), t["dy"].float(), t["x"].dtype
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    xhat, gamma = d * rstd, t["gamma"].float()
    dxhat = dy * gamma
    dx = rstd * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
    return {"y": (xhat * gamma + t["beta"].float()).to(dtype), "stats": torch.cat((mean, rstd), 1), "dx": dx.to(dtype),
            "dgamma": (dy * xhat).sum(0).to(dtype), "dbeta": dy.sum(0).to(dtype)}


def _plain_orthogonal(g, steps):
    """g with its singular values brought near one."""
    x = (g / (torch.linalg.vector_norm(g, dtype=torch.float64) + TINY)).float()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        s = x @ x.t()
        x = A * x + (B * s + C * (s @ s)) @ x
    return x.t() if tall else x


def _plain_muon(c, t):
    g = t["g"].float()
    if c["op"] == "ortho":
        return {"y": _plain_orthogonal(g, c["steps"]).to(t["g"].dtype)}
    t["momentum"].mul_(MU).add_(g)
    o = _plain_orthogonal(g + MU * t["momentum"], c["steps"])
    t["w"].sub_(ALPHA * (o + DECAY * t["w"]))
    return {"w": t["w"], "momentum": t["momentum"]}


def _settings(c, t):
    """Temperature, top_k, top_p and min_p of every row."""
    if c["per_row"]:
        s = t["settings"]
        return s[:, 0].view(torch.float32), s[:, 1], s[:, 2].view(torch.float32), s[:, 3].view(torch.float32)
    like = t["u"]
    return (torch.full_like(like, c["temperature"]), torch.full_like(t["token"], c["top_k"]), torch.full_like(like, c["top_p"]),
            torch.full_like(like, c["min_p"]))


def _plain_sample(c, t):
    """In 64 bits: a random number may lie beside the border of two tokens."""
    x, n, v = t["logits"].double(), c["rows"], c["vocab"]
    temperature, top_k, top_p, min_p = (s[:, None] for s in _settings(c, t))
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = sorted_x[:, :1]
    rank = torch.arange(v, device=x.device)[None, :]
    w = torch.exp((sorted_x - top) / temperature.double())
    keep = (sorted_x > -math.inf) & ((rank < top_k) | (top_k <= 0))
    mass = torch.cumsum(w * keep, 1)
    keep &= (mass - w < top_p.double() * mass[:, -1:]) | (top_p >= 1)
    keep &= w >= min_p.double()
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    # (what the others add to the likeliest token's 1, whose logarithm is that small where one token has it all)
    rest = (w * keep)[:, 1:].sum(1, keepdim=True)
    w = torch.where(kept, torch.exp((x - top) / temperature.double()), torch.zeros((), device=x.device, dtype=torch.float64))
    mass = torch.cumsum(w, 1)
    token = torch.searchsorted(mass, t["u"].double()[:, None] * mass[:, -1:], right=True).clamp(max=v - 1)
    chosen = x.gather(1, token) - top
    logp = chosen - torch.log1p(torch.exp(sorted_x[:, 1:] - top).sum(1, keepdim=True))
    logq = chosen / temperature.double() - torch.log1p(rest)
    return {"token": token[:, 0].to(torch.int32), "kept": kept.sum(1).to(torch.int32), "logp": logp[:, 0].float(), "logq": logq[:, 0].float()}


def _plain_q8(c, t):
    x = t["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127.0
    q = (x / scale).round()  # (to nearest, ties to even)
    z = q @ t["wq"][:, : c["n_in"]].float().t()
    y = z * scale * t["wscale"][None, :]
    return {"y": (y + t["b"].float() if c["bias"] else y).to(t["x"].dtype)}


# ------------------------------------------------------------------------- the library

_library = None


def _tdh():
    global _library
    if _library is None:
        _library = importlib.import_module("tiny-cnn_amd")
        _library.init(torch.cuda.current_device())
    return _library


def _own_run(c, t, b):
    T = _tdh()
    if c["op"] == "norm":
        T.layernorm_fwd(c["rows"], c["len"], b["x"], b["gamma"], b["beta"], b["y"], b["stats"], eps=EPS, dtype=c["dtype"])
        T.layernorm_bwd(c["rows"], c["len"], b["x"], b["gamma"], b["stats"], b["dy"], b["dx"], b["dgamma"], b["dbeta"],
                        dtype=c["dtype"])
        return {k: t[k] for k in ("y", "stats", "dx", "dgamma", "dbeta")}
    if c["op"] == "ortho":
        T.orthogonalize(T.muon_desc(steps=c["steps"], products="f32" if c["dtype"] == "f32" else "f16"), c["rows"], c["cols"],
                        b["g"], b["y"], dtype=c["dtype"])
        return {"y": t["y"]}
    if c["op"] == "muon":
        T.muon_update(T.muon_desc(alpha=ALPHA, mu=MU, lambda_=DECAY, nesterov=True, steps=c["steps"], products="f32"), c["rows"],
                      c["cols"], b["g"], b["w"], b["momentum"], dtype=c["dtype"])
        return {"w": t["w"], "momentum": t["momentum"]}
    if c["op"] == "sample":
        T.sample_tokens(c["rows"], c["vocab"], b["logits"], b["u"], b["token"], logp=b["logp"], logq=b["logq"], kept=b["kept"],
                        temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"],
                        settings=b.get("settings"), dtype=c["dtype"])
        return {k: t[k] for k in ("token", "kept", "logp", "logq")}
    T.fc_q8_fwd(c["n_in"], c["n_out"], c["bias"], c["batch"], b["x"], b["wq"], b["wscale"], b.get("b"), b["y"], dtype=c["dtype"])
    return {"y": t["y"]}


def run(state):
    c, t = state["case"], state["t"]
    if own:
        return _own_run(c, t, state["buf"])
    if c["op"] == "norm":
        return _plain_norm(t)
    return {"muon": _plain_muon, "ortho": _plain_muon, "sample": _plain_sample, "q8": _plain_q8}[c["op"]](c, t)


# --------------------------------------------------------------------------- in 64 bits

def _exact_sample(c, t):
    """Row by row: which tokens are left, and the one whose interval of [0, 1) the random number lies in."""
    out = {"token": [], "kept": [], "logp": [], "logq": []}
    for r in range(c["rows"]):
        if c["per_row"]:
            s = t["settings"][r].cpu().numpy()
            temp, k, p, q = float(s[0:1].view(np.float32)[0]), int(s[1]), float(s[2:3].view(np.float32)[0]), float(s[3:4].view(np.float32)[0])
        else:
            temp, k, p, q = float(np.float32(c["temperature"])), c["top_k"], float(np.float32(c["top_p"])), float(np.float32(c["min_p"]))
        x = t["logits"][r].double()
        fine = torch.nonzero(x > -math.inf)[:, 0]
        order = fine[torch.argsort(-x[fine], stable=True)]  # likeliest first, equal ones by their index
        if k > 0:
            order = order[:k]
        prob = torch.softmax(x[order] / temp, 0)
        if p < 1:
            before = torch.cumsum(prob, 0) - prob
            n = int((before < p).sum())
            order, prob = order[:n], prob[:n]
        n = int((prob >= q * prob[0]).sum())
        ids, _ = torch.sort(order[:n])
        edge = torch.cumsum(torch.softmax(x[ids] / temp, 0), 0)
        at = min(int((edge <= t["u"][r].double() * edge[-1]).sum()), n - 1)
        out["token"].append(ids[at])
        out["kept"].append(torch.tensor(n))
        first = x[order[0]]
        for name, others, scale in (("logq", order[1:n], temp), ("logp", fine[fine != order[0]], 1.0)):
            log_sum = torch.logaddexp(torch.zeros_like(first), torch.logsumexp((x[others] - first) / scale, 0))
            out[name].append((x[ids[at]] - first) / scale - log_sum)
    return {k: torch.stack([v.to("cuda") for v in vs]).to(torch.int32 if k in ("token", "kept") else torch.float64) for k, vs in out.items()}


def exact(case, seed):
    state = prepare(case, seed)
    c, t = state["case"], state["t"]
    if c["op"] == "sample":
        return _exact_sample(c, t)
    d = {k: v.double() for k, v in t.items() if v is not None and k not in ("y", "dx", "stats")}
    if c["op"] == "norm":
        var, mean = torch.var_mean(d["x"], 1, correction=0, keepdim=True)
        std = torch.sqrt(var + EPS)
        xhat = (d["x"] - mean) / std
        g = d["dy"] * d["gamma"]
        n = c["len"]
        return {"y": torch.addcmul(d["beta"][None, :], xhat, d["gamma"][None, :]), "stats": torch.cat((mean, 1 / std), 1),
                "dx": (n * g - g.sum(1, keepdim=True) - xhat * (g * xhat).sum(1, keepdim=True)) / (n * std),
                "dgamma": torch.einsum("rc,rc->c", d["dy"], xhat), "dbeta": d["dy"].sum(0)}
    if c["op"] == "q8":
        x = t["x"].float()
        scale = (x.abs().max(1).values / np.float32(127)).float()  # the scale is a number of 32 bits, and so is the quotient
        q = torch.round(torch.div(x, scale[:, None])).double()
        y = torch.matmul(q, d["wq"][:, : c["n_in"]].t().contiguous()) * (scale.double()[:, None] * d["wscale"])
        return {"y": y + d["b"] if c["bias"] else y}

    def orthogonal(g):
        # p(s) = s (a + s^2 (b + c s^2)) of every singular value, the Gram matrix on the shorter side
        x = g / (g.square().sum().sqrt() + TINY)
        for _ in range(c["steps"]):
            if c["rows"] > c["cols"]:
                m = x.t() @ x
                x = torch.addmm(x, x, C * (m @ m) + B * m, beta=A)
            else:
                m = x @ x.t()
                x = torch.addmm(x, C * (m @ m) + B * m, x, beta=A)
        return x

    if c["op"] == "ortho":
        return {"y": orthogonal(d["g"])}
    mu, alpha, decay = (float(np.float32(v)) for v in (MU, ALPHA, DECAY))
    momentum = mu * d["momentum"] + d["g"]
    return {"w": (1 - alpha * decay) * d["w"] - alpha * orthogonal(d["g"] + mu * momentum), "momentum": momentum}
