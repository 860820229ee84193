"""Cases and plain forms of the operators that serve and train a KDN model around its scan:

* ``step``   one new token per sequence through a whole KDN mixer between its projections (short convolution, key and
             query normalisation, gates, Kalman gain, memory update and readout, gated output norm), against a pool of
             per-sequence states that is updated in place: ``kdn_b200.decode.IsoKDNStep`` / ``DiagKDNStep``
* ``norm``   the norm after a block, its gate, its learned residual scale, the residual sum and the norm before the next
             block: ``kdn_b200.block_norm.block_norm``, forward and with gradients
* ``sample`` the next token of every row of logits under temperature, top-k, top-p and min-p, from given exponential
             random numbers: ``kdn_b200.sampling.sample``

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits; with ``own`` true it calls the
framework.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HEADS, HEAD_DIM = 18, 128  # the framework's benchmark layout: 18 heads of 128 channels, hidden width 2304
NORM_EPS = 1e-5
ISO_OMEGA_MIN, ISO_R_MIN = 0.0, 0.01
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one user alone, token by token: nothing but latency
        step("iso step, 1 sequence", "iso", 1, HEADS, HEAD_DIM, "bf16"),
        # a small server's batch, an odd number of live sequences
        step("diag step, 13 sequences", "diag", 13, HEADS, HEAD_DIM, "bf16"),
        # narrow heads and fp32 activations, as small models and checks run them
        step("diag step, 50 narrow fp32", "diag", 50, 7, 64, "fp32"),
        # a full server's batch: the states' bytes decide
        step("iso step, 256 sequences", "iso", 256, HEADS, HEAD_DIM, "bf16"),
        # the residual sum and next norm between two blocks while a few sequences decode
        norm("norm, 4 decoding rows", 4, HEADS * HEAD_DIM, "bf16", "bf16", False, False, False, False),
        # training at the benchmark's width with every part: sandwich norm, gate and residual scale
        norm("norm training, all parts", 16384, HEADS * HEAD_DIM, "bf16", "bf16", True, True, True, True),
        # training with the residual stream in fp32 and the plain sum, an odd number of tokens
        norm("norm training, fp32 stream", 4099, HEADS * HEAD_DIM, "fp32", "bf16", False, False, False, True),
        # an odd width, fp32 throughout, with the norm after the block
        norm("norm training, odd width", 1000, 1155, "fp32", "fp32", True, False, True, True),
        # one user's next token
        sample("sample, 1 row", 1, 32000, "bf16", "mixed"),
        # a batch whose requests all ask for something else
        sample("sample, 61 mixed rows", 61, 32000, "bf16", "mixed"),
        # fp32 logits of an odd vocabulary, unfiltered: every random number counts
        sample("sample, 24 unfiltered rows", 24, 100003, "fp32", "none"),
        # a large vocabulary and a full server's batch
        sample("sample, 128 large rows", 128, 131072, "bf16", "mixed"),
    ]


def step(name, variant, batch, heads, dim, dtype):
    return {"name": name, "op": "step", "variant": variant, "batch": batch, "heads": heads, "dim": dim, "dtype": dtype}


def norm(name, rows, width, stream, dtype, post, gate, scale, train):
    """post: a norm after the block; gate, scale: the block's output is gated and scaled; train: with gradients."""
    return {"name": name, "op": "norm", "rows": rows, "width": width, "stream": stream, "dtype": dtype, "post": post,
            "gate": gate, "scale": scale, "train": train}


def sample(name, rows, vocab, dtype, filters):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "filters": filters}


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("step", "norm", "sample"))
    if op == "step":
        dim = rng.choice((64, 128, 128))
        heads = rng.randint(1, 24)
        most = min(256, 256 * HEADS * HEAD_DIM ** 2 // (heads * dim * dim))
        case = step("", rng.choice(("iso", "diag")), _log_uniform(rng, 1, most), heads, dim,
                    rng.choice(("bf16", "bf16", "fp32")))
    elif op == "norm":
        width = rng.choice((HEADS * HEAD_DIM, 8 * rng.randint(8, 1000), rng.randint(65, 8000)))
        stream, dtype = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")))
        most = 16384 * HEADS * HEAD_DIM * (1 if dtype == "bf16" and stream == "bf16" else 0.5)
        case = norm("", _log_uniform(rng, 1, int(most // width)), width, stream, dtype, rng.random() < 0.5,
                    rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.6)
    else:
        vocab = rng.choice((32000, _log_uniform(rng, 300, 160000)))
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        most = min(256, 128 * 131072 // vocab // (1 if dtype == "bf16" else 2))
        case = sample("", _log_uniform(rng, 1, most), vocab, dtype, rng.choice(("mixed", "mixed", "none")))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"step": _prepare_step, "norm": _prepare_norm, "sample": _prepare_sample}[case["op"]](case, gen)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _uniform(gen, *shape, low=0.0, high=1.0):
    return torch.rand(*shape, generator=gen, device="cuda") * (high - low) + low


def _prepare_step(case, gen):
    B, H, D, diag = case["batch"], case["heads"], case["dim"], case["variant"] == "diag"
    dt, C = DTYPES[case["dtype"]], 3 * case["heads"] * case["dim"]
    slots = B + 3  # the pool holds a few sequences that do not decode in this step
    rate = torch.exp(_uniform(gen, H * D, low=math.log(0.001), high=math.log(0.1)))
    state = {
        "case": case,
        # the outputs of the block's input projections
        "qkv": _normal(gen, B, C).to(dt),
        "decay_raw": _normal(gen, B, H * D).to(dt),
        "out_gate": _normal(gen, B, H * D).to(dt),
        # the mixer's parameters
        "conv_weight": _uniform(gen, C, 4, low=-0.5, high=0.5),
        "A_log": torch.log(_uniform(gen, H, low=1.0, high=16.0)),
        "dt_bias": rate + torch.log(-torch.expm1(-rate)),
        "norm_weight": 1.0 + 0.1 * _normal(gen, D),
        # the sequences' states
        "memory": 0.2 * _normal(gen, slots, H, D, D),
        "window": _normal(gen, slots, 3, C).to(dt),
        "slots": torch.randperm(slots, generator=gen, device="cuda")[:B].to(torch.int32),
    }
    if diag:
        state["omega_raw"] = _normal(gen, B, H * D).to(dt)
        state["r_raw"] = _normal(gen, B, H).to(dt)
        state["covariance"] = _uniform(gen, slots, H, D, low=0.05, high=1.5)
    else:
        state["omega_r_raw"] = _normal(gen, B, 2 * H).to(dt)
        state["omega_bias"], state["r_bias"] = 0.5 * _normal(gen, H), 0.5 * _normal(gen, H)
        state["covariance"] = _uniform(gen, slots, H, low=0.05, high=1.5)
    return state


def _prepare_norm(case, gen):
    rows, D, st, dt = case["rows"], case["width"], DTYPES[case["stream"]], DTYPES[case["dtype"]]
    state = {
        "case": case,
        "x": (2.0 * _normal(gen, rows, D)).to(st),
        "y": _normal(gen, rows, D).to(dt),
        "weight": 1.0 + 0.1 * _normal(gen, D),
        "post_weight": 1.0 + 0.1 * _normal(gen, D) if case["post"] else None,
        "gate": _normal(gen, rows, D).to(dt) if case["gate"] else None,
        "scale": 0.5 + 0.1 * _normal(gen, D) if case["scale"] else None,
    }
    if case["train"]:
        state["dz"], state["dh"] = _normal(gen, rows, D).to(st), _normal(gen, rows, D).to(dt)
        state["leaves"] = [state[n].requires_grad_(True) for n in ("x", "y", "weight", "post_weight", "gate", "scale")
                           if state[n] is not None]
    return state


def _prepare_sample(case, gen):
    rows, V, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    spread = _uniform(gen, rows, 1, low=1.0, high=4.0)  # flat and peaked distributions
    logits = (spread * _normal(gen, rows, V)).to(dt)
    some = _uniform(gen, rows)
    # a few rows are held to a grammar: most of their vocabulary is masked
    masked = (some < 0.15)[:, None] & (_uniform(gen, rows, V) < 0.95)
    logits.masked_fill_(masked, -math.inf)
    state = {
        "case": case,
        "logits": logits,
        "noise": torch.empty(rows, V, device="cuda").exponential_(generator=gen).clamp_(min=1e-30),
        "temperature": _uniform(gen, rows, low=0.5, high=1.3),
        "top_k": None, "top_p": None, "min_p": None,
    }
    if case["filters"] == "mixed":
        one = lambda: _uniform(gen, rows)  # noqa: E731
        state["temperature"] = torch.where(one() < 0.1, 0.0, state["temperature"])  # greedy requests
        top_k = torch.exp(_uniform(gen, rows, low=0.0, high=math.log(1000.0))).to(torch.int32)
        state["top_k"] = torch.where(one() < 0.4, 0, top_k).to(torch.int32)  # 0: not asked for
        state["top_p"] = torch.where(one() < 0.4, 1.0, _uniform(gen, rows, low=0.5, high=0.99))
        state["min_p"] = torch.where(one() < 0.6, 0.0, _uniform(gen, rows, low=0.001, high=0.1))
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"step": _own_step, "norm": _own_norm, "sample": _own_sample}[op](state)
    return {"step": _plain_step, "norm": _plain_norm, "sample": _plain_sample}[op](state)


def _framework():
    path = os.path.join(os.getcwd(), "kalman-delta-networks_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own_step(s):
    handle = s.get("handle")
    if handle is None:  # a program makes these once: the mixer's weights and the pool of states
        _framework()
        from kdn_b200.decode import DiagKDNStep, IsoKDNStep, KDNState

        shared = dict(conv_weight=s["conv_weight"], A_log=s["A_log"], dt_bias=s["dt_bias"],
                      norm_weight=s["norm_weight"], norm_eps=NORM_EPS)
        if s["case"]["variant"] == "diag":
            step_ = DiagKDNStep(**shared)
        else:
            step_ = IsoKDNStep(**shared, omega_bias=s["omega_bias"], r_bias=s["r_bias"], omega_min=ISO_OMEGA_MIN,
                               r_min=ISO_R_MIN)
        handle = s["handle"] = (step_, KDNState(s["memory"], s["covariance"], s["window"]))
    step_, pool = handle
    if s["case"]["variant"] == "diag":
        y = step_(pool, s["qkv"], s["decay_raw"], s["omega_raw"], s["r_raw"], s["out_gate"], s["slots"])
    else:
        y = step_(pool, s["qkv"], s["decay_raw"], s["omega_r_raw"], s["out_gate"], s["slots"])
    return {"y": y, "memory": pool.memory, "covariance": pool.covariance, "window": pool.window}


def _own_norm(s):
    if "block_norm" not in s:
        _framework()
        from kdn_b200.block_norm import block_norm

        s["block_norm"] = block_norm
    z, h = s["block_norm"](s["x"], s["y"], s["weight"], post_weight=s["post_weight"], gate=s["gate"], scale=s["scale"],
                           eps=NORM_EPS)
    if not s["case"]["train"]:
        return {"z": z, "h": h}
    return {"z": z, "h": h, "grads": torch.autograd.grad((z, h), s["leaves"], (s["dz"], s["dh"]))}


def _own_sample(s):
    if "sample" not in s:
        _framework()
        from kdn_b200.sampling import sample as sample_

        s["sample"] = sample_
    token, prob = s["sample"](s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"],
                              top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "prob": prob}


def _softplus(x):
    return torch.where(x > 20.0, x, torch.log1p(torch.exp(x)))


def _plain_step(s):
    case, idx = s["case"], s["slots"].long()
    B, H, D = case["batch"], case["heads"], case["dim"]
    taps = torch.cat((s["window"][idx], s["qkv"][:, None]), 1)
    conv = (taps.float() * s["conv_weight"].t()).sum(1)
    q, k, v = (conv * torch.sigmoid(conv)).view(B, 3, H, D).unbind(1)
    decay = -torch.exp(s["A_log"])[:, None] * _softplus((s["decay_raw"].float() + s["dt_bias"]).view(B, H, D))
    alpha, P = torch.exp(decay), s["covariance"][idx]
    if case["variant"] == "diag":
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True)).clamp(min=1e-12)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True)).clamp(min=1e-12)
        omega = _softplus(s["omega_raw"].float()).view(B, H, D)
        r = (0.01 + _softplus(s["r_raw"].float()))[..., None]
        prior = alpha * alpha * P + omega
        kappa = prior * k / (r + (prior * k * k).sum(-1, keepdim=True))
        P = prior / (1.0 + D * k * k / r * prior)
        alpha = alpha.clamp(min=1e-6)
    else:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
        omega = ISO_OMEGA_MIN + _softplus(s["omega_r_raw"][:, :H].float() + s["omega_bias"])
        r = ISO_R_MIN + _softplus(s["omega_r_raw"][:, H:].float() + s["r_bias"])
        prior = (alpha * alpha).mean(-1) * P + omega
        kappa = (prior / (r + prior))[..., None] * k
        P = r * prior / (r + prior)
    S = alpha[..., None] * s["memory"][idx]
    delta = v - torch.einsum("bhk,bhkv->bhv", k, S)
    S = S + kappa[..., None] * delta[..., None, :]
    o = D ** -0.5 * torch.einsum("bhk,bhkv->bhv", q, S)
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + NORM_EPS) * s["norm_weight"]
    y = o.reshape(B, H * D) * torch.sigmoid(s["out_gate"].float())
    s["memory"][idx], s["covariance"][idx], s["window"][idx] = S, P, taps[:, 1:]
    return {"y": y.to(s["qkv"].dtype), "memory": s["memory"], "covariance": s["covariance"], "window": s["window"]}


def _plain_norm(s):
    u = s["y"].float()
    if s["post_weight"] is not None:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + NORM_EPS) * s["post_weight"]
    if s["gate"] is not None:
        u = u * torch.sigmoid(s["gate"].float())
    if s["scale"] is not None:
        u = u * s["scale"]
    z = s["x"].float() + u
    h = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + NORM_EPS) * s["weight"]
    z, h = z.to(s["x"].dtype), h.to(s["y"].dtype)
    if not s["case"]["train"]:
        return {"z": z, "h": h}
    return {"z": z, "h": h, "grads": torch.autograd.grad((z, h), s["leaves"], (s["dz"], s["dh"]))}


def _plain_sample(s):
    logits, T = s["logits"].float(), s["temperature"][:, None]
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    sorted_, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    top = sorted_[:, :1]
    e = torch.where(sorted_ == top, 1.0, torch.exp((sorted_ - top) / T))
    total = e.sum(-1, keepdim=True)
    keep = e > 0
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], logits.shape[1])[:, None]
        keep &= torch.arange(logits.shape[1], device=logits.device) < k
    if s["top_p"] is not None:
        ahead = torch.nn.functional.pad(torch.cumsum(e, -1)[:, :-1], (1, 0))
        keep &= ahead < s["top_p"][:, None] * total
    if s["min_p"] is not None:
        keep &= e >= s["min_p"][:, None]
    keep &= T > 0
    keep[:, 0] = True
    score = torch.where(keep, e / s["noise"].gather(1, order), -1.0)
    win = torch.argmax(score, -1, keepdim=True)
    prob = torch.where(T > 0, e.gather(1, win) / total, 1.0)
    empty = top == -math.inf
    token = torch.where(empty, -1, order.gather(1, win))
    return {"token": token[:, 0], "prob": torch.where(empty, 0.0, prob)[:, 0]}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "step":
        B, H, D = case["batch"], case["heads"], case["dim"]
        act, diag = DTYPES[case["dtype"]].itemsize, case["variant"] == "diag"
        state = 2 * B * H * (4 * D * D + 4 * (D if diag else 1) + 9 * D * act)
        tokens = B * H * act * (3 * D + D + (D + 1 if diag else 2) + D + D)
        weights = 4 * (3 * H * D * 4 + H * D + D + 3 * H)
        return {"bytes": state + tokens + weights, "flops": 9 * B * H * D * D}
    if case["op"] == "norm":
        n, st, dt = case["rows"] * case["width"], DTYPES[case["stream"]].itemsize, DTYPES[case["dtype"]].itemsize
        weights = 4 * case["width"] * (1 + case["post"] + case["scale"])
        moved = 2 * st + 2 * dt + (dt if case["gate"] else 0)
        if case["train"]:  # the cotangents come in, the gradients go out
            moved += 2 * st + 2 * dt + (dt if case["gate"] else 0)
        return {"bytes": n * moved + weights * (2 if case["train"] else 1), "flops": n * (30 if case["train"] else 10)}
    n, rows = case["rows"] * case["vocab"], case["rows"]
    # a filter leaves few tokens, and only theirs of the random numbers are needed
    noise = 4 * n if case["filters"] == "none" else 0
    return {"bytes": n * DTYPES[case["dtype"]].itemsize + noise + rows * 28, "flops": 4 * n}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    state = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    return {"step": _exact_step, "norm": _exact_norm, "sample": _exact_sample}[case["op"]](case, state)


def _exact_step(case, s):
    B, H, D = case["batch"], case["heads"], case["dim"]
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    memory, covariance, window = d["memory"].clone(), d["covariance"].clone(), s["window"].clone()
    log1pexp = lambda t: torch.logaddexp(t, torch.zeros_like(t))  # noqa: E731
    y = torch.empty(B, H, D, dtype=torch.float64, device="cuda")
    slots = s["slots"].tolist()
    for b, slot in enumerate(slots):
        mixed = d["conv_weight"][:, 3] * d["qkv"][b]
        for j in range(3):
            mixed = mixed + d["conv_weight"][:, j] * d["window"][slot, j]
        q, k, v = (mixed / (1 + torch.exp(-mixed))).view(3, H, D)
        if case["variant"] == "diag":
            q, k = (t / torch.linalg.vector_norm(t, dim=1, keepdim=True).clamp(min=1e-12) for t in (q, k))
        else:
            q, k = (t / torch.sqrt(torch.linalg.vector_norm(t, dim=1, keepdim=True) ** 2 + 1e-6) for t in (q, k))
        log_alpha = -torch.exp(d["A_log"]).view(H, 1) * log1pexp(d["decay_raw"][b] + d["dt_bias"]).view(H, D)
        P = covariance[slot]
        if case["variant"] == "diag":
            r = 0.01 + log1pexp(d["r_raw"][b]).view(H, 1)
            prior = torch.exp(2 * log_alpha) * P + log1pexp(d["omega_raw"][b]).view(H, D)
            gain = prior * k / (r + torch.linalg.vecdot(prior * k, k).view(H, 1))
            covariance[slot] = 1 / (1 / prior + D * k ** 2 / r)
            log_alpha = log_alpha.clamp(min=math.log(1e-6))
        else:
            r = ISO_R_MIN + log1pexp(d["omega_r_raw"][b, H:] + d["r_bias"])
            prior = torch.exp(2 * log_alpha).sum(1) / D * P
            prior = prior + ISO_OMEGA_MIN + log1pexp(d["omega_r_raw"][b, :H] + d["omega_bias"])
            gain = (prior / (r + prior)).view(H, 1) * k
            covariance[slot] = 1 / (1 / prior + 1 / r)
        kept = memory[slot] * torch.exp(log_alpha).view(H, D, 1)
        miss = v - torch.matmul(k.view(H, 1, D), kept).view(H, D)
        memory[slot] = kept + torch.matmul(gain.view(H, D, 1), miss.view(H, 1, D))
        o = torch.matmul(q.view(H, 1, D), memory[slot]).view(H, D) / math.sqrt(D)
        o = o / torch.sqrt((o ** 2).sum(1, keepdim=True) / D + NORM_EPS) * d["norm_weight"]
        y[b] = o / (1 + torch.exp(-d["out_gate"][b].view(H, D)))
        window[slot, 0], window[slot, 1], window[slot, 2] = s["window"][slot, 1], s["window"][slot, 2], s["qkv"][b]
    return {"y": y.view(B, H * D), "memory": memory, "covariance": covariance, "window": window.double()}


def _exact_norm(case, s):
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    x, y, n = d["x"], d["y"], case["width"]
    one = torch.ones((), dtype=torch.float64, device="cuda")
    post, scale = (one if d[name] is None else d[name] for name in ("post_weight", "scale"))
    opened = one if d["gate"] is None else 1 / (1 + torch.exp(-d["gate"]))
    inv_y = one if d["post_weight"] is None else ((y ** 2).sum(1, keepdim=True) / n + NORM_EPS) ** -0.5
    yhat = y * inv_y
    z = x + scale * opened * yhat * post
    inv_z = ((z ** 2).sum(1, keepdim=True) / n + NORM_EPS) ** -0.5
    zhat = z * inv_z
    out = {"z": z, "h": zhat * d["weight"]}
    if not case["train"]:
        return out
    # the gradients by hand: through a norm, g -> inv (g - unit mean(g unit))
    g = d["dh"] * d["weight"]
    dz = d["dz"] + inv_z * (g - zhat * ((g * zhat).sum(1, keepdim=True) / n))
    du = dz * scale * opened * post
    dy = du if d["post_weight"] is None else inv_y * (du - yhat * ((du * yhat).sum(1, keepdim=True) / n))
    grads = [dz, dy, (d["dh"] * zhat).sum(0)]
    if d["post_weight"] is not None:
        grads.append((dz * scale * opened * yhat).sum(0))
    if d["gate"] is not None:
        grads.append(dz * scale * yhat * post * opened * (1 - opened))
    if d["scale"] is not None:
        grads.append((dz * opened * yhat * post).sum(0))
    return {**out, "grads": tuple(grads)}


def _exact_sample(case, s):
    rows, V = case["rows"], case["vocab"]
    logits = s["logits"].float().cpu().numpy().astype(np.float64)
    noise = s["noise"].cpu().numpy().astype(np.float64)
    per_row = {k: None if s[k] is None else s[k].cpu().numpy().astype(np.float64)
               for k in ("temperature", "top_k", "top_p", "min_p")}
    token, prob = np.full(rows, -1, np.int64), np.zeros(rows)
    for i in range(rows):
        row, top, T = logits[i], logits[i].max(), per_row["temperature"][i]
        if top == -np.inf:
            continue
        first = int(np.argmax(row))
        if T <= 0:
            token[i], prob[i] = first, 1.0
            continue
        weight = np.exp((row - top) / T)
        order = np.argsort(-row, kind="stable")
        limit = V
        if per_row["top_k"] is not None and per_row["top_k"][i] > 0:
            limit = int(per_row["top_k"][i])
        if per_row["top_p"] is not None:
            reached = np.concatenate(([0.0], np.cumsum(weight[order])[:-1]))
            limit = min(limit, int(np.sum(reached < per_row["top_p"][i] * weight.sum())))
        if per_row["min_p"] is not None:
            limit = min(limit, int(np.sum(weight >= per_row["min_p"][i])))
        kept = order[:max(1, limit)]
        token[i] = kept[np.argmax(weight[kept] / noise[i][kept])]
        prob[i] = weight[token[i]] / weight.sum()
    dev = "cuda"
    return {"token": torch.from_numpy(token).to(dev), "prob": torch.from_numpy(prob).to(dev)}
