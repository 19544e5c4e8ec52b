"""Plain 64-bit restatements of the mixture-of-experts operators: routing, the experts' gated
products, the gated residual norm, and their gradients from the formulas.  Test infrastructure
only; everything runs on the CPU."""
from __future__ import annotations

import torch


# ----------------------------------------------------------------------------------- routing

def route_oracle(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=1,
                 renormalize=True, scale=1.0):
    """(weights, ids, scores) in 64 bits, one token at a time; NaN ranks last and the others are told
    apart without it, ties go to the lowest index, a row of -inf scores 0."""
    z = logits.double()
    t, n = z.shape
    if scoring == "softmax":
        top = z.nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")).amax(1, keepdim=True)
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        s = torch.where(total == 0, torch.zeros_like(e), e / total)
        e = torch.where(z == top, torch.ones_like(e), e)  # (infinity minus infinity)
        total = e.nansum(1, keepdim=True)
        rank_by = torch.where(total == 0, e * 0, e / total)
    else:
        s = rank_by = torch.sigmoid(z)
    choice = z if bias is None and groups in (1, top_groups) else rank_by if bias is None else rank_by + bias.double()
    ids = torch.empty(t, top_k, dtype=torch.int64)
    size = n // groups
    for i in range(t):
        c = choice[i].tolist()
        open_ = set(range(n))
        if groups > top_groups:
            best = []
            for g in range(groups):
                part = sorted((float("-inf") if v != v else v for v in c[g * size:(g + 1) * size]), reverse=True)
                best.append((-sum(part[:2]), g))
            kept = [g for _, g in sorted(best)[:top_groups]]
            open_ = {g * size + j for g in kept for j in range(size)}
        rank = sorted(open_, key=lambda e: (c[e] != c[e], -c[e] if c[e] == c[e] else 0.0, e))
        ids[i] = torch.tensor(rank[:top_k])
    w = s.gather(1, ids)
    if renormalize:
        if scoring == "softmax":  # the same ratio without underflow
            zs = z.gather(1, ids)
            m = zs.amax(1, keepdim=True)
            w = torch.exp(zs - torch.where(m == float("-inf"), torch.zeros_like(m), m))
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale, ids, s


def route_gradient_oracle(logits, ids, dweights, scoring, renormalize, scale):
    z, dw = logits.double(), dweights.double() * scale
    s = torch.softmax(z, 1) if scoring == "softmax" else torch.sigmoid(z)
    picked = s.gather(1, ids)
    rest = torch.sigmoid(-z)  # 1 - sigmoid, to its own last place
    if renormalize:
        total = picked.sum(1, keepdim=True)
        r = picked / total
        ds = (dw - (dw * r).sum(1, keepdim=True)) / total
    else:
        ds = dw
    full = torch.zeros_like(s).scatter_(1, ids, ds)
    if scoring == "softmax":
        return s * (full - (full * s).sum(1, keepdim=True))
    return full * s * rest


# -------------------------------------------------------------------------------------- norm

def norm_oracle(y, residual, post, pre, gate, alpha, eps):
    """(h, n, magnitude of h, magnitude of n): the magnitudes add the absolute values of the
    terms, which is what fp32 rounding errors scale with."""
    y, residual, post, pre = (t.double() for t in (y, residual, post, pre))
    g = 1.0 if gate is None else gate.double()
    r1 = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    b = y * r1 * post
    h = alpha * residual + g * b
    r2 = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    mag = (alpha * residual).abs() + (g * b).abs()
    return h, h * r2 * pre, mag, mag * r2 * pre.abs()


def norm_gradient_oracle(y, residual, post, pre, gate, alpha, eps, dh, dn):
    """{name: (gradient, magnitude of its terms)} from the formulas, over 2-D operands."""
    y, residual, post, pre, dh, dn = (t.double() for t in (y, residual, post, pre, dh, dn))
    g = torch.ones(1, 1, dtype=torch.float64) if gate is None else gate.double()
    r1 = (y.square().mean(1, keepdim=True) + eps).rsqrt()
    a = y * r1
    b = a * post
    h = alpha * residual + g * b
    r2 = (h.square().mean(1, keepdim=True) + eps).rsqrt()
    hm = (alpha * residual).abs() + (g * b).abs()
    u = dn * pre
    total = dh + r2 * (u - h * r2 ** 2 * (u * h).mean(1, keepdim=True))
    mag = dh.abs() + r2 * (u.abs() + hm * r2 ** 2 * (u.abs() * hm).mean(1, keepdim=True))
    v, vm = g * total * post, (g * post).abs() * mag
    out = {"y": (r1 * (v - a * (v * a).mean(1, keepdim=True)),
                 r1 * (vm + a.abs() * (vm * a.abs()).mean(1, keepdim=True))),
           "residual": (alpha * total, abs(alpha) * mag),
           "post": ((g * total * a).sum(0), (g.abs() * mag * a.abs()).sum(0)),
           "pre": ((dn * h * r2).sum(0), (dn.abs() * hm * r2).sum(0))}
    if gate is not None:
        dg, dgm = total * b, mag * b.abs()
        if gate.dim() == 1:
            dg, dgm = dg.sum(0), dgm.sum(0)
        elif gate.shape[1] == 1 and y.shape[1] != 1:
            dg, dgm = dg.sum(1, keepdim=True), dgm.sum(1, keepdim=True)
        out["gate"] = (dg, dgm)
    return out


# ----------------------------------------------------------------------------------- experts

def _act(g, activation):
    """(value, derivative) of the gate's activation."""
    s = torch.sigmoid(g)
    if activation == "silu":
        return g * s, s * (1 + g * (1 - s))
    if activation == "sigmoid":
        return s, s * (1 - s)
    return g, torch.ones_like(g)


def experts_oracle(x, w12, w3, ids, weights, activation="silu", dy=None):
    """y, and with ``dy`` the gradients (y, dx, dw12, dw3, dweights), expert by expert.  Slots whose
    id is not an expert contribute nothing."""
    x, w = x.double(), weights.double()
    y = torch.zeros(x.shape[0], w3.shape[2], dtype=torch.float64)
    if dy is not None:
        dy = dy.double()
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        dw12, dw3 = torch.zeros(w12.shape, dtype=torch.float64), torch.zeros(w3.shape, dtype=torch.float64)
    for e in range(w12.shape[0]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if not token.numel():
            continue
        a, b, weight = w12[e].double(), w3[e].double(), w[token, slot].unsqueeze(1)
        gu = x[token] @ a
        act, slope = _act(gu[:, 0::2], activation)
        up = gu[:, 1::2]
        h = act * up
        o = h @ b
        y.index_add_(0, token, weight * o)
        if dy is not None:
            dout = weight * dy[token]
            dh = dout @ b.t()
            dgu = torch.stack((dh * up * slope, dh * act), 2).flatten(1)
            dw[token, slot] = (dy[token] * o).sum(1)
            dw3[e] = h.t() @ dout
            dw12[e] = x[token].t() @ dgu
            dx.index_add_(0, token, dgu @ a.t())
    return y if dy is None else (y, dx, dw12, dw3, dw)
