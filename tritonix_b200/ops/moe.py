"""Mixture-of-experts layers: routing tokens to experts and the experts' gated products.

``route_experts`` turns router logits into the experts each token uses and their weights;
``moe_swiglu`` is ``swiglu_mlp`` with many expert MLPs of which each token uses a few; ``moe_block``
joins them with the norms around a block (ops/norm.py).  All have their gradients.  The reference
has no counterpart.
"""
from __future__ import annotations

import ctypes

import torch

from tritonix_b200 import _cabi
from tritonix_b200.ops.norm import gated_residual_norm


_route_problems: dict = {}


def _route(logits, bias, problem):
    shape = (logits.shape[0], problem.top_k)
    weights = torch.empty(shape, device=logits.device, dtype=torch.float32)
    ids = torch.empty(shape, device=logits.device, dtype=torch.int32)
    _cabi.call(logits.device, _cabi.lib.tnx_route_experts, ctypes.byref(problem), logits.data_ptr(),
               bias.data_ptr() if bias is not None else None, weights.data_ptr(), ids.data_ptr())
    return weights, ids


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, problem):
        weights, ids = _route(logits, bias, problem)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, ids)
        ctx.problem = problem
        ctx.mark_non_differentiable(ids)
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return None, None, None
        logits, ids = ctx.saved_tensors
        return _route_backward(dweights, logits, ids, ctx.problem), None, None


def _route_backward(dweights, logits, ids, problem):
    dweights = dweights.contiguous()
    dlogits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    _cabi.call(logits.device, _cabi.lib.tnx_route_experts_backward, ctypes.byref(problem), logits.data_ptr(),
               ids.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
    return dlogits


def route_gradient(dweights, logits, ids, scoring, renormalize, scale):
    """Gradient of the logits from that of the weights (the custom operator's backward pass)."""
    logits = _cabi.rows_view(logits)
    problem = _check_route(logits, ids.shape[1], scoring, None, 1, 1, renormalize, scale)
    return _route_backward(dweights, logits, ids.contiguous(), problem)


def route_experts(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax",
                  bias: torch.Tensor | None = None, num_groups: int = 1, top_groups: int = 1,
                  renormalize: bool = True, scale: float = 1.0):
    """Returns ``(weights, ids)``, both [tokens, top_k]: fp32 weights and int32 expert numbers, best
    expert first.

    ``logits`` [tokens, experts] in fp16, bf16 or fp32, at most 512 experts.  Scores are the softmax
    or the sigmoid (``scoring``) of the logits; experts are chosen by score + ``bias`` (fp32
    [experts]; it balances the load, takes no part in the weights and has no gradient), ties going
    to the lowest index.  With ``num_groups`` > 1 only experts of the ``top_groups`` groups of
    consecutive experts whose two best choices have the largest sum can be chosen.  The weights are
    the chosen experts' scores, divided by their sum if ``renormalize``, times ``scale``.

    Experts are told apart as in 64-bit arithmetic, however close.  An expert whose logit is -inf
    has the score 0 (a row of nothing else has the weights 0).  A NaN logit ranks last, and the other
    experts are told apart as if it were not there; a softmax that is not renormalised still gives
    its token NaN weights.  ``ids`` are always distinct and in range."""
    _cabi.refuse_tangents(logits)
    top_k, num_groups, top_groups = int(top_k), int(num_groups), int(top_groups)
    renormalize, scale = bool(renormalize), _cabi.number("scale", scale)
    key = (_cabi.signature(logits, bias), top_k, scoring, num_groups, top_groups, renormalize, scale)
    problem = _route_problems.get(key)
    if problem is None:
        problem = _cabi.remember(_route_problems, key, _check_route(logits, top_k, scoring, bias, num_groups, top_groups,
                                                                    renormalize, scale))
    if not problem.stride_logits:
        logits = _cabi.rows_view(logits)
        return route_experts(logits, top_k, scoring=scoring, bias=bias, num_groups=num_groups, top_groups=top_groups,
                             renormalize=renormalize, scale=scale)
    if bias is not None:
        bias = bias.detach().contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteExperts.apply(logits, bias, problem)
    return _route(logits, bias, problem)


def _check_route(logits, top_k, scoring, bias, groups, top_groups, renormalize, scale) -> _cabi.RouteProblem:
    """The C problem of a call whose arguments are sound; its stride is 0 where the logits have to be
    copied first."""
    _cabi.require_cuda(logits, *([bias] if bias is not None else []))
    if logits.dim() != 2 or logits.dtype not in _cabi.DTYPES:
        raise ValueError("logits must be a 2-D float16, bfloat16 or float32 tensor, got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    if scoring not in _cabi.SCORINGS:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if bias is not None:
        if tuple(bias.shape) != (logits.shape[1],) or bias.dtype != torch.float32:
            raise ValueError(f"bias must be a float32 tensor of {logits.shape[1]} elements, got "
                             f"{tuple(bias.shape)} {bias.dtype}")
        if bias.device != logits.device:
            raise ValueError("logits and bias must live on the same device")
    if logits.shape[0] >= 1 << 31:
        raise ValueError("too many tokens")
    stride = max(logits.stride(0), logits.shape[1]) if logits.shape[0] <= 1 else logits.stride(0)
    if _cabi.rows_view(logits) is not logits:
        stride = 0
    return _cabi.RouteProblem(logits.shape[0], logits.shape[1], top_k, groups, top_groups,
                              _cabi.SCORINGS[scoring], int(renormalize), _cabi.DTYPES[logits.dtype], scale, 0, stride)


# ------------------------------------------------------------------------------ experts' products

_MAX_EXPERTS = 512


def _addressable(t: torch.Tensor) -> bool:
    """Adjacent elements in rows, pitches of 16 bytes, no overlapping rows or matrices."""
    fine, extent = t.stride(-1) == 1, t.shape[-1]
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size > 1:
            fine = fine and step % 8 == 0 and step >= extent
        extent = size * (step if size > 1 else extent)
    return fine


def _pitched(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the copy engine can address it: itself, or a contiguous copy."""
    fine = _addressable(t) and t.data_ptr() % 16 == 0
    return t if fine else t.clone(memory_format=torch.contiguous_format)


def _pitches(t: torch.Tensor) -> list:
    """Strides of all dimensions but the last, from the first on; those of dimensions of one element
    (torch may give any) as if it were contiguous."""
    out, extent = [], t.shape[-1]
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        step = step if size > 1 else extent
        out.append(step)
        extent = step * size
    return out[::-1]


class _MoePlan:
    """What a call signature needs, worked out once: the C problem and its resources without and with
    gradients, or that operands have to be copied first."""

    def __init__(self, x, w12, w3, ids, weights, activation):
        act = _check_moe(x, w12, w3, ids, weights, activation)
        self.addressable = all(_addressable(t) for t in (x, w12, w3))
        if not self.addressable:
            return
        self.out = (x.shape[0], w3.shape[2])
        self.pairs, self.device = ids.shape, x.device
        (sx,), (s12e, s12k), (s3e, s3k) = _pitches(x), _pitches(w12), _pitches(w3)
        self.problems, self.resources = [], []
        for train in (0, 1):
            problem = _cabi.MoeProblem(x.shape[0], w12.shape[0], ids.shape[1], x.shape[1], w3.shape[1], w3.shape[2],
                                       _cabi.DTYPES[x.dtype], act, int(ids.dtype == torch.int64), train, sx, s12e, s12k,
                                       s3e, s3k, w3.shape[2])
            res = _cabi.MoeResources()
            _cabi.raise_for(_cabi.lib.tnx_moe_query(ctypes.byref(problem), ctypes.byref(res)))
            self.problems.append(problem)
            self.resources.append(res)


_moe_plans: dict = {}


def _moe_forward(plan, x, w12, w3, ids, weights, train):
    device = plan.device
    y = torch.empty(plan.out, device=device, dtype=x.dtype)
    # (scratch of the call's own: calls on different streams or in different graphs never share it)
    nbytes = plan.resources[train].workspace_bytes
    workspace = torch.empty(nbytes, device=device, dtype=torch.uint8)
    saved = torch.empty(plan.resources[1].saved_bytes, device=device, dtype=torch.uint8) if train else None
    _cabi.call(device, _cabi.lib.tnx_moe_swiglu, ctypes.byref(plan.problems[train]), x.data_ptr(), w12.data_ptr(),
               w3.data_ptr(), ids.data_ptr(), weights.data_ptr(), y.data_ptr(), saved.data_ptr() if train else None,
               workspace.data_ptr(), nbytes, _cabi.status_word(device).data_ptr())
    return y, saved


class _MoeSwiglu(torch.autograd.Function):
    """Keeps the operands, the pairs' order, the hidden activation (16 bits) and the gate/up products
    (fp32): 10 bytes per pair and hidden column."""

    @staticmethod
    def forward(ctx, x, w12, w3, weights, ids, plan):
        y, saved = _moe_forward(plan, x, w12, w3, ids, weights, 1)
        ctx.save_for_backward(x, w12, w3, saved)
        ctx.plan = plan
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return *_moe_backward(ctx.plan, dy, *ctx.saved_tensors, ctx.needs_input_grad[:4]), None, None


def _moe_backward(plan, dy, x, w12, w3, saved, wants):
    """Gradients of x, w12, w3 and the weights; None where not wanted."""
    dy = _pitched(dy)
    (stride_dy,) = _pitches(dy)
    new = lambda shape, dtype: torch.empty(shape, device=x.device, dtype=dtype)  # noqa: E731
    dx = new(x.shape, x.dtype) if wants[0] else None
    dw12 = new(w12.shape, x.dtype) if wants[1] else None
    dw3 = new(w3.shape, x.dtype) if wants[2] else None
    dweights = new(plan.pairs, torch.float32) if wants[3] else None
    workspace = new(plan.resources[1].backward_workspace_bytes, torch.uint8)
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    _cabi.call(x.device, _cabi.lib.tnx_moe_swiglu_backward, ctypes.byref(plan.problems[1]), dy.data_ptr(), stride_dy,
               x.data_ptr(), w12.data_ptr(), w3.data_ptr(), saved.data_ptr(), ptr(dx), ptr(dw12), ptr(dw3),
               ptr(dweights), workspace.data_ptr(), workspace.numel(), _cabi.status_word(x.device).data_ptr())
    return dx, dw12, dw3, dweights


def moe_swiglu(x: torch.Tensor, w12: torch.Tensor, w3: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
               activation: str = "silu") -> torch.Tensor:
    """The experts' MLPs of every token, weighted and added:

        y[t] = sum over slots s of  weights[t, s] * ((act(x[t] W1[e]) * (x[t] W2[e])) W3[e]),  e = ids[t, s]

    ``x`` [tokens, D]; ``w12`` [experts, D, 2F], each expert's W1 and W2 column-interleaved
    (``interleave_weights``); ``w3`` [experts, F, N]: all fp16 or all bf16, with D, F and N multiples
    of 8 and at most 512 experts.  ``ids`` [tokens, top_k] int32 or int64 and ``weights`` fp32, as
    ``route_experts`` returns them; a slot whose id is not an expert (-1, say) contributes nothing,
    and an expert may stand in several slots of a token.  ``activation``: "silu", "sigmoid" or
    "none" (``swiglu`` and ``glu`` take the same).

    The hidden activation, times its weight, is rounded to the operands' type between the two products
    (not for a single token without gradients).  A call's scratch is 4 bytes per (token, slot) pair and column of ``y``, times
    up to eight where there are few tiles, and 2 per pair and column of ``x`` and of the hidden
    activation; training keeps 10 per pair and hidden column.

    Gradients flow to ``x``, ``w12``, ``w3`` and ``weights``.  The routing stays on the device: no
    call waits for it.  Results do not depend on timing (every sum has a fixed order)."""
    _cabi.refuse_tangents(x, w12, w3, weights)
    key = (_cabi.signature(x, w12, w3, ids, weights), activation)
    plan = _moe_plans.get(key)
    if plan is None:
        plan = _cabi.remember(_moe_plans, key, _MoePlan(x, w12, w3, ids, weights, activation))
    if not plan.addressable or (x.data_ptr() | w12.data_ptr() | w3.data_ptr()) & 15:
        return moe_swiglu(_pitched(x), _pitched(w12), _pitched(w3), ids, weights, activation)
    ids, weights = ids.contiguous(), weights.contiguous()
    if (x.requires_grad or w12.requires_grad or w3.requires_grad or weights.requires_grad) \
            and torch.is_grad_enabled():
        return _MoeSwiglu.apply(x, w12, w3, weights, ids, plan)
    return _moe_forward(plan, x, w12, w3, ids, weights, 0)[0]


# The two passes of moe_swiglu as the custom operators call them: with operands of any strides, what is
# kept between the passes in a tensor of its own.

def _moe_plan(x, w12, w3, ids, weights, activation):
    x, w12, w3 = _pitched(x), _pitched(w12), _pitched(w3)
    return x, w12, w3, _MoePlan(x, w12, w3, ids, weights, activation)


def moe_forward_kept(x, w12, w3, ids, weights, activation):
    _check_moe(x, w12, w3, ids, weights, activation)
    x, w12, w3, plan = _moe_plan(x, w12, w3, ids, weights, activation)
    return _moe_forward(plan, x, w12, w3, ids.contiguous(), weights.contiguous(), 1)


def moe_gradients_kept(dy, x, w12, w3, ids, saved, activation, wants):
    weights = torch.empty(ids.shape, device=ids.device, dtype=torch.float32)  # (for the checks: `saved` has them)
    x, w12, w3, plan = _moe_plan(x, w12, w3, ids, weights, activation)
    return _moe_backward(plan, dy, x, w12, w3, saved, wants)


def moe_saved_bytes(x, w12, w3, ids, activation) -> int:
    """Size of what a training forward call keeps, from shapes alone."""
    (n, d, two_f), n_out = map(int, w12.shape), int(w3.shape[2])
    problem = _cabi.MoeProblem(int(x.shape[0]), n, int(ids.shape[1]), d, two_f // 2, n_out, _cabi.DTYPES[x.dtype],
                               _cabi.ACTIVATIONS[activation], int(ids.dtype == torch.int64), 1, d, d * two_f, two_f,
                               two_f // 2 * n_out, n_out, n_out)
    res = _cabi.MoeResources()
    _cabi.raise_for(_cabi.lib.tnx_moe_query(ctypes.byref(problem), ctypes.byref(res)))
    return res.saved_bytes


def _check_moe(x, w12, w3, ids, weights, activation) -> int:
    _cabi.require_cuda(x, w12, w3, ids, weights)
    if x.dtype not in (torch.float16, torch.bfloat16) or w12.dtype != x.dtype or w3.dtype != x.dtype:
        raise ValueError(f"x, w12 and w3 must all be float16 or all bfloat16, got {x.dtype}, {w12.dtype}, {w3.dtype}")
    if x.dim() != 2 or w12.dim() != 3 or w3.dim() != 3:
        raise ValueError("moe_swiglu expects x (tokens, D), w12 (experts, D, 2F) and w3 (experts, F, N)")
    if w12.shape[0] != w3.shape[0] or w12.shape[1] != x.shape[1] or w12.shape[2] != 2 * w3.shape[1]:
        raise ValueError(f"shapes do not fit: x {tuple(x.shape)}, w12 {tuple(w12.shape)}, w3 {tuple(w3.shape)}")
    # (the library's own limits, refused here because operands of other sizes have no pitch that the
    # copy engine can address, however they are copied)
    if not 1 <= w12.shape[0] <= _MAX_EXPERTS:
        raise ValueError(f"1 to {_MAX_EXPERTS} experts, got {w12.shape[0]}")
    if any(size < 8 or size % 8 for size in (x.shape[1], w3.shape[1], w3.shape[2])):
        raise ValueError("d_model, d_ff and n_out must be positive multiples of 8, got "
                         f"{x.shape[1]}, {w3.shape[1]}, {w3.shape[2]}")
    if ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.shape[1] < 1 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be int32 or int64 (tokens, top_k), got {tuple(ids.shape)} {ids.dtype}")
    if weights.shape != ids.shape or weights.dtype != torch.float32:
        raise ValueError(f"weights must be float32 {tuple(ids.shape)}, got {tuple(weights.shape)} {weights.dtype}")
    if any(t.device != x.device for t in (w12, w3, ids, weights)):
        raise ValueError("all operands must live on the same device")
    act = _cabi.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_cabi.ACTIVATIONS)}, got {activation!r}")
    return act


# ---------------------------------------------------------------------------------- the whole block

def moe_block(x: torch.Tensor, residual: torch.Tensor, logits: torch.Tensor, w12: torch.Tensor, w3: torch.Tensor,
              post_weight: torch.Tensor, pre_weight: torch.Tensor, top_k: int, *, scoring: str = "softmax",
              bias: torch.Tensor | None = None, num_groups: int = 1, top_groups: int = 1, renormalize: bool = True,
              scale: float = 1.0, activation: str = "silu", gate: torch.Tensor | None = None,
              residual_scale: float = 1.0, eps: float = 1e-6):
    """A mixture-of-experts block from its normalised input to the next block's:

        weights, ids = route_experts(logits, top_k, ...)
        y = moe_swiglu(x, w12, w3, ids, weights, activation)
        h, n = gated_residual_norm(y, residual, post_weight, pre_weight, gate, residual_scale, eps)

    ``x`` [tokens, D] is the block's input, ``logits`` [tokens, experts] its router's output (``matmul``
    of ``x`` and the router's weights, say), ``residual`` [tokens, N] the residual stream; the other
    arguments are those of the three operators.  Returns ``(h, n)``: the new residual stream and the
    next block's input.  Gradients flow through all of it."""
    weights, ids = route_experts(logits, top_k, scoring=scoring, bias=bias, num_groups=num_groups,
                                 top_groups=top_groups, renormalize=renormalize, scale=scale)
    y = moe_swiglu(x, w12, w3, ids, weights, activation)
    return gated_residual_norm(y, residual, post_weight, pre_weight, gate, residual_scale, eps)
