"""Measured cases of the mixture-of-experts operators: routing, the experts' SwiGLU products and
the gated residual norm between two blocks.

Each case names one operator (``op``), its sizes and types, and whether the backward pass runs.
``run`` computes it in plain torch operations, or with ``own = True`` through tritonix_b200.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------- cases

def _route(tokens, experts, top_k, dtype, scoring="softmax", bias=False, groups=1, top_groups=1,
           renormalize=True, train=False):
    return {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "scoring": scoring, "bias": bias, "groups": groups, "top_groups": top_groups,
            "renormalize": renormalize, "train": train}


def _experts(tokens, experts, top_k, d_model, d_ff, dtype, train=False):
    return {"op": "experts", "tokens": tokens, "experts": experts, "top_k": top_k,
            "d_model": d_model, "d_ff": d_ff, "dtype": dtype, "train": train}


def _norm(tokens, d_model, dtype, weights="fp32", gate="channel", train=False):
    return {"op": "norm", "tokens": tokens, "d_model": d_model, "dtype": dtype,
            "weights": weights, "gate": gate, "train": train}


def listed():
    return [
        # one token being generated: nothing but latency
        {"name": "route token", **_route(1, 64, 8, "bf16")},
        # a prompt batch on a model with many experts in groups, balanced by a bias
        {"name": "route prompt grouped", **_route(32768, 256, 8, "fp32", "sigmoid", True, 8, 4)},
        # a training step's router, an odd number of tokens after packing
        {"name": "route train", **_route(16383, 64, 6, "fp32", train=True)},
        # one token being generated through its eight experts
        {"name": "experts token", **_experts(1, 64, 8, 2048, 1024, "bf16")},
        # a small batch of sequences being generated: nearly every expert is read for a few rows
        {"name": "experts decode batch", **_experts(33, 64, 8, 2048, 1024, "bf16")},
        # a short prompt through eight experts of the size of this repository's MLP benchmark
        {"name": "experts wide prompt", **_experts(500, 8, 2, 4096, 14336, "fp16")},
        # a long prompt batch, compute bound
        {"name": "experts prompt", **_experts(8192, 64, 8, 2048, 1024, "bf16")},
        # a training step, forward and backward, sizes that fill no tile
        {"name": "experts train", **_experts(4095, 16, 4, 2048, 2040, "bf16", True)},
        # the seam between two blocks for one token
        {"name": "norm token", **_norm(1, 4096, "bf16", "bf16")},
        # the same for a prompt batch
        {"name": "norm prompt", **_norm(32768, 4096, "bf16", "bf16")},
        # a training step with 32-bit weights and a gate of each token's own
        {"name": "norm train", **_norm(16383, 4096, "bf16", "fp32", "channel", True)},
        # a wide 32-bit residual stream of an odd width, gated element by element
        {"name": "norm train full gate", **_norm(2047, 5001, "fp32", "fp32", "full", True)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "norm"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.randint(max(2, 8 // groups), 256 // groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(10, top_groups * (experts // groups)))
        return _route(_log(rng, 1, 32768), experts, top_k, rng.choice(["bf16", "fp16", "fp32"]),
                      rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups,
                      # (one expert renormalised is the constant 1: its gradient is nothing to compare)
                      top_k > 1 and rng.random() < 0.7, rng.random() < 0.4)
    if op == "norm":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case = _norm(_log(rng, 1, 32768), _log(rng, 64, 8192), dtype, rng.choice([dtype, "fp32"]),
                     rng.choice(["none", "channel", "token", "full"]), rng.random() < 0.5)
        limit = max(work(c)["bytes"] for c in listed() if c["op"] == "norm")
    else:
        experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
        case = _experts(_log(rng, 1, 8192), experts, rng.randint(1, min(8, experts)),
                        8 * _log(rng, 32, 512), 8 * _log(rng, 32, 512),
                        rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.4)
        while 6 * experts * case["d_model"] * case["d_ff"] > 3 << 30:  # bytes of the weights
            case["d_ff"] = 8 * (case["d_ff"] // 16)
        limit = max(work(c)["flops"] for c in listed() if c["op"] == "experts")
    key = "bytes" if op == "norm" else "flops"
    while work(case)[key] > limit:
        case["tokens"] = case["tokens"] * 3 // 4
    return case


def work(case):
    t = case["tokens"]
    if case["op"] == "route":
        n, size = case["experts"], _BYTES[case["dtype"]]
        # logits in, weights and ids out; the backward pass reads the weights' gradient (and what
        # the forward pass read and wrote) and writes the logits' gradient
        moved = t * n * size + t * case["top_k"] * 8 + (4 * n if case["bias"] else 0)
        if case["train"]:
            moved += t * n * size + t * case["top_k"] * 4
        return {"bytes": moved, "flops": 4 * t * n}
    d = case["d_model"]
    if case["op"] == "norm":
        size, wsize = _BYTES[case["dtype"]], _BYTES[case["weights"]]
        gate = {"none": 0, "channel": d * wsize, "token": t * wsize, "full": t * d * wsize}[case["gate"]]
        moved = 4 * t * d * size + 2 * d * wsize + gate
        if case["train"]:  # two gradients in, those of block, residual, weights and gate out
            moved += 4 * t * d * size + 2 * d * wsize + gate
        return {"bytes": moved, "flops": (40 if case["train"] else 12) * t * d}
    f, pairs, size = case["d_ff"], t * case["top_k"], _BYTES[case["dtype"]]
    used = min(case["experts"], pairs)
    moved = 3 * used * d * f * size + 2 * t * d * size + pairs * 8
    flops = 6 * pairs * d * f
    if case["train"]:  # gradients of x, of the routing weights and of every expert's weights
        moved += 3 * case["experts"] * d * f * size + 2 * t * d * size + pairs * 4
        flops *= 3
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, scale, generator=g)

    t, train = case["tokens"], case["train"]
    state = {"case": case}
    if case["op"] == "route":
        n, k = case["experts"], case["top_k"]
        # logits of a trained router: a token's own preferences over experts of unequal popularity
        logits = (normal(t, n, scale=1.5) + normal(n, scale=0.7)).to(_TYPES[case["dtype"]])
        state["logits"] = logits.requires_grad_(train)
        state["bias"] = normal(n, scale=0.05) if case["bias"] else None
        state["grad"] = normal(t, k) if train else None
        return state
    d, dtype = case["d_model"], _TYPES[case["dtype"]]
    if case["op"] == "norm":
        wtype = _TYPES[case["weights"]]
        # a residual stream that has grown over many blocks, with a few loud channels
        loud = 1.0 + 8.0 * (torch.rand(d, device="cuda", generator=g) < 0.01)
        state["y"] = normal(t, d).to(dtype)
        state["residual"] = (normal(t, d, scale=3.0) * loud).to(dtype)
        state["post"] = (1.0 + normal(d, scale=0.1)).to(wtype)
        state["pre"] = (1.0 + normal(d, scale=0.1)).to(wtype)
        shape = {"none": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[case["gate"]]
        state["gate"] = None if shape is None else (0.5 + normal(*shape, scale=0.2)).to(wtype)
        if train:
            for name in ("y", "residual", "post", "pre", "gate"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
            state["grads"] = [normal(t, d).to(dtype), normal(t, d).to(dtype)]
        return state
    n, k, f = case["experts"], case["top_k"], case["d_ff"]
    state["x"] = normal(t, d).to(dtype)
    state["w12"] = normal(n, d, 2 * f, scale=d ** -0.5, dtype=dtype)
    state["w3"] = normal(n, f, d, scale=f ** -0.5, dtype=dtype)
    logits = normal(t, n) + normal(n, scale=0.3)
    top = logits.topk(k, dim=1)
    state["ids"] = top.indices.to(torch.int32)
    state["weights"] = torch.softmax(top.values, dim=1)
    if train:
        for name in ("x", "w12", "w3", "weights"):
            state[name].requires_grad_(True)
        state["grad"] = normal(t, d).to(dtype)
    return state


# ------------------------------------------------------------------------------- plain forms

def _route_plain(logits, bias, case):
    # in 64 bits: experts whose scores are next to each other have to come in the right order
    t, n = logits.shape
    z = logits.double()
    if case["scoring"] == "softmax":
        e = torch.exp(z - z.detach().max(1, keepdim=True).values)
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-z))
    choice = score.detach() if bias is None else score.detach() + bias.double()
    groups = case["groups"]
    if groups > 1:
        best = choice.view(t, groups, -1).sort(2, descending=True).values[:, :, :2].sum(2)
        kept = best.argsort(dim=1, descending=True, stable=True)[:, :case["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = choice.masked_fill(~open_.repeat_interleave(n // groups, 1), -math.inf)
    ids = choice.argsort(dim=1, descending=True, stable=True)[:, :case["top_k"]]
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return weights.float(), ids.to(torch.int32)


def _experts_plain(x, w12, w3, ids, weights):
    t, k = ids.shape
    n, d, f2 = w12.shape
    flat = ids.reshape(-1).long()
    if t * k <= n:  # few tokens: each with its own copy of its experts' weights
        rows = x.float().repeat_interleave(k, 0).unsqueeze(1)
        gu = torch.bmm(rows, w12[flat].float())
        h = gu[..., 0::2] / (1.0 + torch.exp(-gu[..., 0::2])) * gu[..., 1::2]
        out = torch.bmm(h, w3[flat].float()).squeeze(1)
    else:  # rows sorted by expert, each expert's rows filled up to the longest
        order = flat.argsort(dim=0, stable=True)
        count = torch.bincount(flat, minlength=n)
        most = int(count.max())
        rank = torch.arange(t * k, device=x.device) - (count.cumsum(0) - count)[flat[order]]
        place = flat[order] * most + rank
        rows = x.new_zeros((n * most, d), dtype=torch.float32).index_copy(0, place, x.float()[order // k])
        gu = torch.bmm(rows.view(n, most, d), w12.float())
        h = gu[..., 0::2] / (1.0 + torch.exp(-gu[..., 0::2])) * gu[..., 1::2]
        done = torch.bmm(h, w3.float()).view(n * most, -1)[place]
        out = torch.zeros_like(done).index_copy(0, order, done)
    return (out.view(t, k, -1) * weights.unsqueeze(2)).sum(1).to(x.dtype)


def _norm_plain(y, residual, post, pre, gate):
    yf = y.float()
    a = yf * torch.rsqrt((yf * yf).mean(1, keepdim=True) + 1e-6) * post.float()
    h = 0.5 * residual.float() + (a if gate is None else a * gate.float())
    n = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * pre.float()
    return h.to(residual.dtype), n.to(residual.dtype)


def run(state):
    case, train = state["case"], state["case"]["train"]
    if own:
        import tritonix_b200 as tritonix
    if case["op"] == "route":
        logits, bias = state["logits"], state["bias"]
        if own:
            weights, ids = tritonix.route_experts(
                logits, case["top_k"], scoring=case["scoring"], bias=bias,
                num_groups=case["groups"], top_groups=case["top_groups"],
                renormalize=case["renormalize"])
        else:
            weights, ids = _route_plain(logits, bias, case)
        out = {"weights": weights, "ids": ids}
        if train:
            out["grad_logits"] = torch.autograd.grad(weights, logits, state["grad"])[0]
        return out
    if case["op"] == "norm":
        args = [state[name] for name in ("y", "residual", "post", "pre", "gate")]
        if own:
            h, n = tritonix.gated_residual_norm(*args, residual_scale=0.5, eps=1e-6)
        else:
            h, n = _norm_plain(*args)
        out = {"h": h, "n": n}
        if train:
            leaves = [a for a in args if a is not None]
            out["grads"] = torch.autograd.grad([h, n], leaves, state["grads"])
        return out
    args = [state[name] for name in ("x", "w12", "w3", "ids", "weights")]
    y = tritonix.moe_swiglu(*args) if own else _experts_plain(*args)
    out = {"y": y}
    if train:
        leaves = [state[name] for name in ("x", "w12", "w3", "weights")]
        out["grads"] = torch.autograd.grad(y, leaves, state["grad"])
    return out


# ------------------------------------------------------------------------------ in 64 bits

def _route_exact(state):
    case, z = state["case"], state["logits"].detach().double()
    t, n = z.shape
    p = torch.softmax(z, 1) if case["scoring"] == "softmax" else torch.sigmoid(z)
    left = p if state["bias"] is None else p + state["bias"].double()
    index = torch.arange(n, device=z.device).expand(t, n)
    groups = case["groups"]
    if groups > 1:
        size = n // groups
        top = left.view(t, groups, size).topk(min(2, size), dim=2).values.sum(2)
        group = torch.arange(groups, device=z.device)
        # a group's place: how many groups are better, or as good with a lower index
        better = (top[:, None, :] > top[:, :, None]) | (
            (top[:, None, :] == top[:, :, None]) & (group[None, None, :] < group[None, :, None]))
        shut = better.sum(2) >= case["top_groups"]
        left = torch.where(shut.repeat_interleave(size, 1), -math.inf, left)
    picks = []
    for _ in range(case["top_k"]):
        best = left.max(1, keepdim=True).values
        pick = torch.where(left == best, index, n).min(1, keepdim=True).values
        picks.append(pick)
        left = left.scatter(1, pick, -math.inf)
    ids = torch.cat(picks, 1)
    s = p.gather(1, ids)
    total = s.sum(1, keepdim=True) if case["renormalize"] else torch.ones_like(s[:, :1])
    w = s / total
    out = {"weights": w, "ids": None}
    if case["train"]:
        dw = state["grad"].double()
        ds = (dw - (dw * w).sum(1, keepdim=True)) / total if case["renormalize"] else dw
        dp = torch.zeros_like(p).scatter(1, ids, ds)
        if case["scoring"] == "softmax":
            out["grad_logits"] = p * (dp - (dp * p).sum(1, keepdim=True))
        else:
            out["grad_logits"] = dp * p * (1.0 - p)
    return out


def _norm_exact(state):
    y, res, post, pre = (state[name].detach().double() for name in ("y", "residual", "post", "pre"))
    gate = 1.0 if state["gate"] is None else state["gate"].detach().double()
    r1 = 1.0 / torch.sqrt((y * y).mean(1, keepdim=True) + 1e-6)
    b = y * r1 * post
    h = 0.5 * res + gate * b
    r2 = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)
    out = {"h": h, "n": h * r2 * pre}
    if state["case"]["train"]:
        dh, dn = (v.double() for v in state["grads"])
        u = dn * pre
        dh = dh + r2 * (u - h * r2 * r2 * (u * h).mean(1, keepdim=True))
        db = gate * dh
        u = db * post
        dy = r1 * (u - y * r1 * r1 * (u * y).mean(1, keepdim=True))
        grads = [dy, 0.5 * dh, (db * y * r1).sum(0), (dn * h * r2).sum(0)]
        if state["gate"] is not None:
            dg = dh * b
            form = state["case"]["gate"]
            grads.append(dg.sum(0) if form == "channel" else dg.sum(1, keepdim=True) if form == "token" else dg)
        out["grads"] = grads
    return out


def _experts_exact(state):
    x, w = state["x"].detach().double(), state["weights"].detach().double()
    ids, train = state["ids"].long(), state["case"]["train"]
    w12, w3 = state["w12"].detach(), state["w3"].detach()
    y = torch.zeros(x.shape[0], w3.shape[2], dtype=torch.float64, device=x.device)
    if train:
        dy = state["grad"].double()
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        dw12, dw3 = (torch.zeros(v.shape, dtype=torch.float64, device=x.device) for v in (w12, w3))
    for e in range(w12.shape[0]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if not token.numel():
            continue
        up_gate, down, weight = w12[e].double(), w3[e].double(), w[token, slot].unsqueeze(1)
        gu = x[token] @ up_gate
        gate, up = gu[:, 0::2], gu[:, 1::2]
        s = torch.sigmoid(gate)
        h = gate * s * up
        o = h @ down
        y.index_add_(0, token, weight * o)
        if train:
            dw[token, slot] = (dy[token] * o).sum(1)
            dout = weight * dy[token]
            dh = dout @ down.t()
            dgu = torch.stack((dh * up * s * (1.0 + gate * (1.0 - s)), dh * gate * s), 2).flatten(1)
            dw3[e] = h.t() @ dout
            dw12[e] = x[token].t() @ dgu
            dx.index_add_(0, token, dgu @ up_gate.t())
    return {"y": y, "grads": [dx, dw12, dw3, dw]} if train else {"y": y}


def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _route_exact, "norm": _norm_exact, "experts": _experts_exact}[case["op"]](state)
