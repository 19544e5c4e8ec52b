"""Mixture-of-experts layers: routing tokens to experts and the experts' gated products.

``route_experts`` turns router logits into the experts each token uses and their weights, with a
gradient for the logits.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes

import torch

from tritonix_b200 import _cabi


def _route_problem(logits, top_k, groups, top_groups, scoring, renormalize, scale):
    return _cabi.RouteProblem(logits.shape[0], logits.shape[1], top_k, groups, top_groups, scoring,
                              int(renormalize), _cabi.DTYPES[logits.dtype], scale, 0, logits.stride(0))


def _route(logits, bias, args):
    problem = _route_problem(logits, *args)
    shape = (logits.shape[0], args[0])
    weights = torch.empty(shape, device=logits.device, dtype=torch.float32)
    ids = torch.empty(shape, device=logits.device, dtype=torch.int32)
    _cabi.call(logits.device, _cabi.lib.tnx_route_experts, ctypes.byref(problem), logits.data_ptr(),
               bias.data_ptr() if bias is not None else None, weights.data_ptr(), ids.data_ptr())
    return weights, ids


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, args):
        weights, ids = _route(logits, bias, args)
        ctx.save_for_backward(logits, ids)
        ctx.args = args
        ctx.mark_non_differentiable(ids)
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _):
        logits, ids = ctx.saved_tensors
        problem = _route_problem(logits, *ctx.args)
        dweights = dweights.contiguous()
        dlogits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        _cabi.call(logits.device, _cabi.lib.tnx_route_experts_backward, ctypes.byref(problem),
                   logits.data_ptr(), ids.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
        return dlogits, None, None


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
    has the score 0 (a row of nothing else has the weights 0); a NaN logit ranks last.  ``ids`` are
    always distinct and in range."""
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
        bias = bias.detach().contiguous()
    logits = _cabi.rows_view(logits)
    args = (int(top_k), int(num_groups), int(top_groups), _cabi.SCORINGS[scoring], bool(renormalize),
            float(scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteExperts.apply(logits, bias, args)
    return _route(logits, bias, args)
