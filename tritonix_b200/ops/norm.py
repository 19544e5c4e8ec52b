"""The seam between two transformer blocks, forward and backward, one kernel each.

``gated_residual_norm`` takes the output of the block that has just finished (``swiglu_mlp``,
``moe_swiglu``, an attention block) and the residual stream it was computed from, and returns the
new residual stream with the next block's input:

    h = residual_scale * residual + gate * rms(y) * post_weight
    n = rms(h) * pre_weight                      rms(v) = v / sqrt(mean(v^2) + eps) over a row

A row is read once; sums are fp32, and ``n`` is computed from ``h`` before ``h`` is rounded to the
output type.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes

import torch

from tritonix_b200 import _cabi

_MAX_COLS = 16384


def _gate_form(gate, rows: int, cols: int, lead) -> int:
    """How the gate is laid out, from its shape: a value per channel, per token or per element."""
    if gate is None:
        return _cabi.GATE_NONE
    shape = tuple(gate.shape)
    # (a single row's [cols] is a channel gate; a single column's [rows, 1] a token gate)
    if shape == (cols,):
        return _cabi.GATE_CHANNEL
    if shape == (*lead, 1):
        return _cabi.GATE_TOKEN
    if shape == (*lead, cols):
        return _cabi.GATE_FULL
    raise ValueError(f"gate must be {(cols,)}, {(*lead, 1)} or {(*lead, cols)}, got {shape}")


def _problem(rows, cols, dtype, weight_dtype, form, residual_scale, eps, y, residual, gate):
    return _cabi.NormProblem(rows, cols, _cabi.DTYPES[dtype], _cabi.DTYPES[weight_dtype], form,
                             residual_scale, eps, 0, y.stride(0), residual.stride(0),
                             gate.stride(0) if form in (_cabi.GATE_TOKEN, _cabi.GATE_FULL) else 0)


def _forward(y, residual, post, pre, gate, form, residual_scale, eps, keep_stats):
    rows, cols = y.shape
    h = torch.empty((rows, cols), device=y.device, dtype=y.dtype)
    n = torch.empty_like(h)
    stats = torch.empty((rows, 2), device=y.device, dtype=torch.float32) if keep_stats else None
    problem = _problem(rows, cols, y.dtype, post.dtype, form, residual_scale, eps, y, residual, gate)
    _cabi.call(y.device, _cabi.lib.tnx_gated_residual_norm, ctypes.byref(problem), y.data_ptr(),
               residual.data_ptr(), post.data_ptr(), pre.data_ptr(),
               gate.data_ptr() if gate is not None else None, h.data_ptr(), n.data_ptr(),
               stats.data_ptr() if stats is not None else None)
    return h, n, stats


class _GatedResidualNorm(torch.autograd.Function):
    """Over 2-D operands.  Keeps y, residual and two reciprocal norms per row."""

    @staticmethod
    def forward(ctx, y, residual, post, pre, gate, form, residual_scale, eps):
        h, n, stats = _forward(y, residual, post, pre, gate, form, residual_scale, eps, True)
        ctx.save_for_backward(y, residual, post, pre, gate, stats)
        ctx.args = (form, residual_scale, eps)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        y, residual, post, pre, gate, stats = ctx.saved_tensors
        form, residual_scale, eps = ctx.args
        rows, cols = y.shape
        dh, dn = _cabi.rows_view(dh), _cabi.rows_view(dn)
        problem = _problem(rows, cols, y.dtype, post.dtype, form, residual_scale, eps, y, residual, gate)
        dy = torch.empty((rows, cols), device=y.device, dtype=y.dtype)
        dres = torch.empty_like(dy)
        dpost, dpre = (torch.empty(cols, device=y.device, dtype=post.dtype) for _ in range(2))
        dgate = None
        if gate is not None:
            dgate = torch.empty(gate.shape, device=y.device, dtype=gate.dtype)
        nbytes = _cabi.lib.tnx_gated_residual_norm_workspace(ctypes.byref(problem))
        workspace = torch.empty(max(nbytes, 16), device=y.device, dtype=torch.uint8)
        _cabi.call(y.device, _cabi.lib.tnx_gated_residual_norm_backward, ctypes.byref(problem),
                   dh.data_ptr(), dh.stride(0), dn.data_ptr(), dn.stride(0), y.data_ptr(),
                   residual.data_ptr(), post.data_ptr(), pre.data_ptr(),
                   gate.data_ptr() if gate is not None else None, stats.data_ptr(), dy.data_ptr(),
                   dres.data_ptr(), dpost.data_ptr(), dpre.data_ptr(),
                   dgate.data_ptr() if dgate is not None else None, workspace.data_ptr(),
                   workspace.numel())
        return dy, dres, dpost, dpre, dgate, None, None, None


def gated_residual_norm(y: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                        pre_weight: torch.Tensor, gate: torch.Tensor | None = None,
                        residual_scale: float = 1.0, eps: float = 1e-6):
    """Returns ``(h, n)``: the new residual stream and the next block's normalised input.

    ``y`` and ``residual``: [..., D] of one type (fp16, bf16, fp32), D <= 16384.  ``post_weight``,
    ``pre_weight``: [D], and ``gate``: [D] (per channel), [..., 1] (per token) or [..., D] (per
    element), all of one type: that of ``y`` or fp32.  Gradients flow to every tensor argument;
    rows need not be contiguous with one another."""
    tensors = [t for t in (y, residual, post_weight, pre_weight, gate) if t is not None]
    _cabi.require_cuda(*tensors)
    if y.dtype not in _cabi.DTYPES or residual.dtype != y.dtype:
        raise ValueError(f"y and residual must share one of float16, bfloat16, float32; got {y.dtype}, "
                         f"{residual.dtype}")
    if y.dim() < 1 or residual.shape != y.shape:
        raise ValueError(f"y and residual must have the same shape, got {tuple(y.shape)}, {tuple(residual.shape)}")
    lead, cols = tuple(y.shape[:-1]), y.shape[-1]
    if not 1 <= cols <= _MAX_COLS:
        raise ValueError(f"rows must have 1 to {_MAX_COLS} elements, got {cols}")
    if tuple(post_weight.shape) != (cols,) or tuple(pre_weight.shape) != (cols,):
        raise ValueError(f"post_weight and pre_weight must be {(cols,)}, got {tuple(post_weight.shape)}, "
                         f"{tuple(pre_weight.shape)}")
    wtype = post_weight.dtype
    if wtype not in (y.dtype, torch.float32) or any(t.dtype != wtype for t in (pre_weight, gate) if t is not None):
        raise ValueError(f"the weights and the gate must share one type, {y.dtype} or float32")
    if any(t.device != y.device for t in tensors):
        raise ValueError("all operands must live on the same device")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps}")
    rows = y.numel() // cols
    if rows >= 1 << 31:
        raise ValueError("too many rows")
    form = _gate_form(gate, rows, cols, lead)
    y2, r2 = _cabi.rows_view(y.reshape(rows, cols)), _cabi.rows_view(residual.reshape(rows, cols))
    post, pre = post_weight.contiguous(), pre_weight.contiguous()
    if form == _cabi.GATE_CHANNEL:
        gate = gate.contiguous()
    elif form != _cabi.GATE_NONE:
        gate = _cabi.rows_view(gate.reshape(rows, gate.shape[-1]))
        if gate.stride(0) < 0:
            gate = gate.contiguous()
    args = (y2, r2, post, pre, gate, form, float(residual_scale), float(eps))
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        h, n = _GatedResidualNorm.apply(*args)
    else:
        h, n, _ = _forward(*args, False)
    return h.view(y.shape), n.view(y.shape)
