"""The dense operators that sit next to the grouped GEMMs of a mixture-of-experts layer, as measured cases.

* ``gated``: the gated feed-forward block of a shared or dense expert, ``act(x Wg^T) * (x Wu^T)``, and its backward pass;
* ``linear``: the projection behind it, ``act(x W^T + b) + residual``, and its backward pass;
* ``router``: the gate in front of the experts, the top-k choice with its weights, and its backward pass.

``run`` computes a case in plain torch operations, or, with ``own`` set, through ``cudnn_frontend_b200``.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # serving: one new token through a wide dense expert
        {"name": "gated_one_token", "op": "gated", "dir": "fwd", "m": 1, "k": 4096, "i": 14336, "act": "swiglu", "type": "bf16", "pad": 0, "save": False},
        # serving: a small decode batch through a shared expert
        {"name": "gated_decode_batch", "op": "gated", "dir": "fwd", "m": 25, "k": 7168, "i": 2048, "act": "geglu", "type": "fp16", "pad": 0, "save": False},
        # training: the forward pass of a dense expert over a long batch, with what its backward pass reads
        {"name": "gated_train_forward", "op": "gated", "dir": "fwd", "m": 8192, "k": 4096, "i": 14336, "act": "swiglu", "type": "bf16", "pad": 0, "save": True},
        # training: the backward pass of a dense expert
        {"name": "gated_train_backward", "op": "gated", "dir": "bwd", "m": 4096, "k": 4096, "i": 14336, "act": "swiglu", "type": "bf16", "pad": 0},
        # training: a ragged batch of a shared expert
        {"name": "gated_ragged_backward", "op": "gated", "dir": "bwd", "m": 1531, "k": 7168, "i": 2048, "act": "geglu", "type": "fp16", "pad": 64},
        # serving: the down projection of a few new tokens onto the residual stream
        {"name": "linear_decode_batch", "op": "linear", "dir": "fwd", "m": 7, "k": 14336, "n": 4096, "act": "", "bias": False, "residual": True, "type": "bf16", "out": "bf16", "pad": 0, "save": False},
        # prefill: the down projection of a long prompt onto the residual stream
        {"name": "linear_prefill", "op": "linear", "dir": "fwd", "m": 8192, "k": 14336, "n": 4096, "act": "", "bias": False, "residual": True, "type": "bf16", "out": "bf16", "pad": 0, "save": False},
        # odd sizes: everything in the epilogue at once
        {"name": "linear_odd_epilogue", "op": "linear", "dir": "fwd", "m": 777, "k": 1000, "n": 2001, "act": "gelu", "bias": True, "residual": True, "type": "fp16", "out": "fp16", "pad": 24, "save": True},
        # training: a projection with an activation and a bias
        {"name": "linear_train_backward", "op": "linear", "dir": "bwd", "m": 4096, "k": 4096, "n": 14336, "act": "silu", "bias": True, "type": "bf16", "out": "bf16", "pad": 0},
        # training: the router's projection, whose gradient arrives in 32 bits
        {"name": "linear_router_backward", "op": "linear", "dir": "bwd", "m": 8192, "k": 7168, "n": 256, "act": "", "bias": False, "type": "bf16", "out": "fp32", "pad": 0},
        # training: 8 of 256 experts by biased sigmoid scores, forward and backward
        {"name": "router_train", "op": "router", "dir": "both", "t": 32768, "e": 256, "topk": 8, "score": "sigmoid", "normalize": True, "bias": True, "masked": False, "type": "fp32"},
        # serving: 2 of 8 experts for a decode batch
        {"name": "router_decode_batch", "op": "router", "dir": "fwd", "t": 64, "e": 8, "topk": 2, "score": "softmax", "normalize": True, "bias": False, "masked": False, "type": "fp32"},
    ]


def _between(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["gated", "gated", "linear", "linear", "router"])
    if op == "router":
        e = _between(rng, 4, 512)
        return {"op": op, "dir": rng.choice(["fwd", "both"]), "t": _between(rng, 1, 32768), "e": e, "topk": rng.randint(1, min(e, 16)),
                "score": rng.choice(["softmax", "sigmoid"]), "normalize": rng.random() < 0.7, "bias": rng.random() < 0.4, "masked": rng.random() < 0.3,
                "type": rng.choice(["fp32", "fp32", "bf16", "fp16"])}  # fmt: skip
    most = max(work(c)["flops"] for c in listed())
    while True:
        c = {"op": op, "dir": rng.choice(["fwd", "fwd", "bwd"]), "m": _between(rng, 1, 8192), "k": _between(rng, 64, 14336, 8),
             "type": rng.choice(["bf16", "bf16", "fp16"]), "pad": rng.choice([0, 0, 8, 64])}  # fmt: skip
        save = rng.random() < 0.5 and c["dir"] == "fwd"
        if op == "gated":
            c |= {"i": _between(rng, 64, 14336), "act": rng.choice(["swiglu", "geglu"])}
        else:
            c |= {"n": _between(rng, 8, 14336), "act": rng.choice(["", "relu", "silu", "gelu"]), "bias": rng.random() < 0.5}
            c["out"] = "fp32" if not c["act"] and rng.random() < 0.25 else c["type"]
            if c["dir"] == "fwd":
                c["residual"] = rng.random() < 0.5
        if c["dir"] == "fwd":
            c["save"] = save and bool(c["act"])
        if work(c)["flops"] <= most:
            return c


def _rows(shape, dtype, pad, gen):
    """Normal values [rows, cols], as a view into rows that are `pad` values longer."""
    return torch.randn((shape[0], shape[1] + pad), dtype=torch.float32, device="cuda", generator=gen).to(dtype)[:, : shape[1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    dt = _TYPES[case["type"]]
    if case["op"] == "router":
        t, e = case["t"], case["e"]
        logits = 1.5 * torch.randn((t, e), device="cuda", generator=gen)
        if case["masked"]:  # experts that are switched off for some rows, and now and then all of them
            off = torch.rand((t, e), device="cuda", generator=gen) < 0.3
            off |= torch.rand((t, 1), device="cuda", generator=gen) < 0.02
            logits = logits.masked_fill(off, -math.inf)
        s["logits"] = logits.to(dt)
        s["bias"] = 0.05 * torch.randn((e,), device="cuda", generator=gen) if case["bias"] else None
        s["dweights"] = torch.randn((t, case["topk"]), device="cuda", generator=gen)
        return s
    m, k = case["m"], case["k"]
    s["x"] = _rows((m, k), dt, case["pad"], gen)
    if case["op"] == "gated":
        i = case["i"]
        size = (2.5 if case["act"] == "geglu" else 1.0) / math.sqrt(k)  # wide enough for GeGLU's limits to be met
        s["w_gate"] = (size * torch.randn((i, k), device="cuda", generator=gen)).to(dt)
        s["w_up"] = (size * torch.randn((i, k), device="cuda", generator=gen)).to(dt)
        if case["dir"] == "bwd":
            s["dh"] = torch.randn((m, i), device="cuda", generator=gen).to(dt)
            s["gate"] = (s["x"].float() @ s["w_gate"].float().t()).to(dt)
            s["up"] = (s["x"].float() @ s["w_up"].float().t()).to(dt)
        return s
    n = case["n"]
    s["weight"] = (torch.randn((n, k), device="cuda", generator=gen) / math.sqrt(k)).to(dt)
    s["bias"] = torch.randn((n,), device="cuda", generator=gen).to(dt) if case["bias"] else None
    if case["dir"] == "bwd":
        s["dy"] = torch.randn((m, n), device="cuda", generator=gen).to(_TYPES[case["out"]])
        s["preact"] = None
        if case["act"]:
            z = s["x"].float() @ s["weight"].float().t()
            s["preact"] = (z + s["bias"].float() if case["bias"] else z).to(dt)
    else:
        s["residual"] = torch.randn((m, n), device="cuda", generator=gen).to(dt) if case["residual"] else None
    return s


def run(state):
    if own:
        return _run_own(state)
    return {"gated": _plain_gated, "linear": _plain_linear, "router": _plain_router}[state["case"]["op"]](state)


def _run_own(s):
    import cudnn_frontend_b200 as cf

    c = s["case"]
    if c["op"] == "gated":
        if c["dir"] == "fwd":
            return cf.gated_ffn(s["x"], s["w_gate"], s["w_up"], act_func=c["act"], return_preact=c["save"])
        return cf.gated_ffn_backward(s["dh"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"], act_func=c["act"])
    if c["op"] == "linear":
        if c["dir"] == "fwd":
            return cf.linear(s["x"], s["weight"], bias=s["bias"], act_func=c["act"] or None, residual=s["residual"], out_dtype=_TYPES[c["out"]],
                             return_preact=c["save"])  # fmt: skip
        return cf.linear_backward(s["dy"], s["x"], s["weight"], preact=s["preact"], act_func=c["act"] or None, bias_grad=c["bias"])
    how = {"score_func": c["score"], "normalize": c["normalize"], "scale": 2.5}
    weights, ids = cf.router_topk(s["logits"], c["topk"], bias=s["bias"], **how)
    if c["dir"] == "fwd":
        return weights, ids
    return weights, ids, cf.router_topk_backward(s["dweights"], s["logits"], ids, **how)


# ---- plain forms: 32 bits (64 for the router's biased scores, whose order decides), rounded once ----


def _glu(gate, up, act):
    if act == "geglu":
        gate, up = gate.clamp(max=7.0), up.clamp(-7.0, 7.0) + 1.0
        return gate * torch.sigmoid(1.702 * gate) * up
    return gate * torch.sigmoid(gate) * up


def _glu_grads(dh, gate, up, act):
    """Gradients of `_glu` with respect to gate and up."""
    if act == "geglu":
        g, u = gate.clamp(max=7.0), up.clamp(-7.0, 7.0) + 1.0
        sig = torch.sigmoid(1.702 * g)
        dgate = dh * u * sig * (1.0 + 1.702 * g * (1.0 - sig)) * (gate <= 7.0)
        return dgate, dh * g * sig * (up.abs() <= 7.0)
    sig = torch.sigmoid(gate)
    return dh * up * sig * (1.0 + gate * (1.0 - sig)), dh * gate * sig


def _plain_gated(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    if c["dir"] == "fwd":
        gate, up = x @ wg.t(), x @ wu.t()
        h = _glu(gate, up, c["act"]).to(dt)
        return (h, gate.to(dt), up.to(dt)) if c["save"] else h
    dgate, dup = _glu_grads(s["dh"].float(), s["gate"].float(), s["up"].float(), c["act"])
    return (dgate @ wg + dup @ wu).to(dt), (dgate.t() @ x).to(dt), (dup.t() @ x).to(dt)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0.0).to(z.dtype)
    if act == "silu":
        sig = torch.sigmoid(z)
        return sig * (1.0 + z * (1.0 - sig))
    return 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    if c["dir"] == "fwd":
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        y = y.to(_TYPES[c["out"]])
        return (y, z.to(dt)) if c["save"] else y
    dz = s["dy"].float()
    if c["act"]:
        dz = dz * _act_grad(s["preact"].float(), c["act"])
    return (dz @ w).to(dt), (dz.t() @ x).to(dt), dz.sum(0) if c["bias"] else None


def _plain_router(s):
    c, logits = s["case"], s["logits"].float()
    order = logits
    if s["bias"] is not None:
        wide = logits.double()
        score = torch.sigmoid(wide) if c["score"] == "sigmoid" else _softmax(wide, -1)
        order = (score + s["bias"].double()).masked_fill(logits == -math.inf, -math.inf)
    top, ids = torch.sort(order, dim=1, descending=True, stable=True)  # ties go to the lowest index
    ids = ids[:, : c["topk"]]
    chosen = logits.gather(1, ids)
    there = top[:, : c["topk"]] > -math.inf
    if c["score"] == "sigmoid":
        weights = _softmax(_log_sigmoid(chosen), 1) if c["normalize"] else torch.sigmoid(chosen)
    elif c["normalize"]:
        weights = _softmax(chosen, 1)
    else:
        weights = _softmax(logits, 1).gather(1, ids)
    weights = 2.5 * weights.masked_fill(~there, 0.0)
    told = ids.masked_fill(~there, -1).to(torch.int32)
    if c["dir"] == "fwd":
        return weights, told
    dw = s["dweights"].masked_fill(~there, 0.0)
    if c["normalize"]:
        grads = weights * (dw - (weights * dw).sum(1, keepdim=True) / 2.5)
        if c["score"] == "sigmoid":
            grads = grads * torch.sigmoid(-chosen)
    elif c["score"] == "sigmoid":
        grads = dw * weights * torch.sigmoid(-chosen)
    else:
        grads = dw * weights
    grads = torch.zeros_like(logits).scatter(1, ids, grads.masked_fill(~there, 0.0))
    if c["score"] == "softmax" and not c["normalize"]:
        grads = grads - _softmax(logits, 1) * grads.sum(1, keepdim=True)
    return weights, told, grads.to(s["logits"].dtype)


def _softmax(v, dim):
    """Over what is above -inf; 0 where nothing is."""
    e = torch.exp(v - v.amax(dim, keepdim=True).clamp(min=torch.finfo(v.dtype).min))
    return e / e.sum(dim, keepdim=True).clamp(min=torch.finfo(v.dtype).tiny)


def _log_sigmoid(v):
    return v.clamp(max=0.0) - torch.log1p(torch.exp(-v.abs()))


def work(case):
    if case["op"] == "router":
        size = 4 if case["type"] == "fp32" else 2
        t, e, k = case["t"], case["e"], case["topk"]
        read, flops = t * e * size + t * k * 8 + (4 * e if case["bias"] else 0), 4 * t * e
        if case["dir"] == "both":
            read, flops = read + t * e * size + t * k * 4, 2 * flops
        return {"bytes": read, "flops": flops}
    m, k = case["m"], case["k"]
    if case["op"] == "gated":
        i = case["i"]
        if case["dir"] == "fwd":
            return {"bytes": 2 * (m * k + 2 * i * k + (3 if case["save"] else 1) * m * i), "flops": 4 * m * i * k}
        return {"bytes": 2 * (3 * m * i + 2 * m * k + 4 * i * k), "flops": 8 * m * i * k}
    n, out = case["n"], 4 if case["out"] == "fp32" else 2
    if case["dir"] == "fwd":
        extra = (2 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0) + (2 * m * n if case["save"] else 0)
        return {"bytes": 2 * (m * k + n * k) + out * m * n + extra, "flops": 2 * m * n * k}
    extra = (4 * n if case["bias"] else 0) + (2 * m * n if case["act"] else 0)
    return {"bytes": out * m * n + 2 * (2 * m * k + 2 * n * k) + extra, "flops": 4 * m * n * k}


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits; the router's choice is a whole number and has none."""
    s = prepare(case, seed)
    f = {name: v.double() for name, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "gated":
        if case["dir"] == "fwd":
            gate, up = torch.einsum("mk,ik->mi", f["x"], f["w_gate"]), torch.einsum("mk,ik->mi", f["x"], f["w_up"])
        else:
            gate, up = f["gate"].requires_grad_(), f["up"].requires_grad_()
        if case["act"] == "geglu":
            g = torch.where(gate > 7, torch.full_like(gate, 7), gate)
            u = torch.where(up > 7, torch.full_like(up, 7), torch.where(up < -7, torch.full_like(up, -7), up))
            h = (u + 1) * g / (1 + torch.exp(-1.702 * g))
        else:
            h = up * gate / (1 + torch.exp(-gate))
        if case["dir"] == "fwd":
            return (h, gate, up) if case["save"] else h
        dgate, dup = torch.autograd.grad(h, (gate, up), f["dh"])
        dx = torch.einsum("mi,ik->mk", dgate, f["w_gate"]) + torch.einsum("mi,ik->mk", dup, f["w_up"])
        return dx, torch.einsum("mi,mk->ik", dgate, f["x"]), torch.einsum("mi,mk->ik", dup, f["x"])
    if case["op"] == "linear":
        if case["dir"] == "fwd":
            z = torch.einsum("mk,nk->mn", f["x"], f["weight"]) + f.get("bias", 0.0)
        else:
            z = f["preact"].requires_grad_() if case["act"] else None
        if case["act"] == "relu":
            a = torch.where(z > 0, z, torch.zeros_like(z))
        elif case["act"] == "silu":
            a = z / (1 + torch.exp(-z))
        elif case["act"] == "gelu":
            a = z * (1 + torch.erf(z / math.sqrt(2.0))) / 2
        else:
            a = z
        if case["dir"] == "fwd":
            y = a + f.get("residual", 0.0)
            return (y, z) if case["save"] else y
        dz = torch.autograd.grad(a, z, f["dy"])[0] if case["act"] else f["dy"]
        return torch.einsum("mn,nk->mk", dz, f["weight"]), torch.einsum("mn,mk->nk", dz, f["x"]), dz.sum(0) if case["bias"] else None
    logits = f["logits"].requires_grad_()
    on = logits > -math.inf
    safe = torch.where(on, logits, torch.zeros_like(logits))
    score = 1 / (1 + torch.exp(-safe))
    if case["score"] == "softmax":
        e = torch.exp(safe - safe.detach().amax(1, keepdim=True)) * on
        score = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    order = (score if case["bias"] else safe).detach() + f.get("bias", 0.0)
    order = torch.where(on, order, torch.full_like(order, -math.inf))
    at = torch.argsort(order, dim=1, descending=True, stable=True)[:, : case["topk"]]
    chosen = score.gather(1, at) * on.gather(1, at)
    weights = 2.5 * (chosen / chosen.sum(1, keepdim=True).clamp(min=1e-300) if case["normalize"] else chosen)
    if case["dir"] == "fwd":
        return weights.detach(), None
    (dlogits,) = torch.autograd.grad(weights, logits, f["dweights"])
    return weights.detach(), None, dlogits
