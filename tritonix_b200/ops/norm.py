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


class _NormPlan:
    """What a call signature needs, worked out once: the C problem for operands as rows, or that they
    have to be brought into that shape first."""

    def __init__(self, y, residual, post, pre, gate, residual_scale, eps):
        form = _check(y, residual, post, pre, gate, eps)
        rows, cols = y.numel() // y.shape[-1], y.shape[-1]
        parts = [y, residual] + ([gate] if form in (_cabi.GATE_TOKEN, _cabi.GATE_FULL) else [])
        vectors = [post, pre] + ([gate] if form == _cabi.GATE_CHANNEL else [])
        self.ready = all(t.dim() == 2 and _cabi.rows_view(t) is t for t in parts) and \
            all(t.is_contiguous() for t in vectors)
        self.form, self.shape = form, (rows, cols)
        if not self.ready:
            return
        pitch = lambda t: t.stride(0) if rows > 1 else t.shape[1]  # noqa: E731
        self.problem = _cabi.NormProblem(rows, cols, _cabi.DTYPES[y.dtype], _cabi.DTYPES[post.dtype], form,
                                         residual_scale, eps, 0, pitch(y), pitch(residual),
                                         pitch(gate) if len(parts) == 3 else 0)
        self.workspace_bytes = max(_cabi.lib.tnx_gated_residual_norm_workspace(ctypes.byref(self.problem)), 16)


_plans: dict = {}


def _forward(plan, y, residual, post, pre, gate, keep_stats):
    h = torch.empty(plan.shape, device=y.device, dtype=y.dtype)
    n = torch.empty_like(h)
    stats = torch.empty((plan.shape[0], 2), device=y.device, dtype=torch.float32) if keep_stats else None
    _cabi.call(y.device, _cabi.lib.tnx_gated_residual_norm, ctypes.byref(plan.problem), y.data_ptr(),
               residual.data_ptr(), post.data_ptr(), pre.data_ptr(),
               gate.data_ptr() if gate is not None else None, h.data_ptr(), n.data_ptr(),
               stats.data_ptr() if stats is not None else None, _cabi.status_word(y.device).data_ptr())
    return h, n, stats


class _GatedResidualNorm(torch.autograd.Function):
    """Over 2-D operands.  Keeps y, residual and two reciprocal norms per row."""

    @staticmethod
    def forward(ctx, y, residual, post, pre, gate, plan):
        h, n, stats = _forward(plan, y, residual, post, pre, gate, True)
        ctx.save_for_backward(y, residual, post, pre, gate, stats)
        ctx.plan = plan
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        return *_backward(ctx.plan, dh, dn, *ctx.saved_tensors), None


def _backward(plan, dh, dn, y, residual, post, pre, gate, stats):
    device = y.device
    dh, dn = _cabi.rows_view(dh), _cabi.rows_view(dn)
    dy = torch.empty(plan.shape, device=device, dtype=y.dtype)
    dres = torch.empty_like(dy)
    dpost, dpre = torch.empty((2, plan.shape[1]), device=device, dtype=post.dtype).unbind()
    dgate = torch.empty(gate.shape, device=device, dtype=gate.dtype) if gate is not None else None
    workspace = torch.empty(plan.workspace_bytes, device=device, dtype=torch.uint8)
    _cabi.call(device, _cabi.lib.tnx_gated_residual_norm_backward, ctypes.byref(plan.problem),
               dh.data_ptr(), dh.stride(0), dn.data_ptr(), dn.stride(0), y.data_ptr(),
               residual.data_ptr(), post.data_ptr(), pre.data_ptr(),
               gate.data_ptr() if gate is not None else None, stats.data_ptr(), dy.data_ptr(),
               dres.data_ptr(), dpost.data_ptr(), dpre.data_ptr(),
               dgate.data_ptr() if dgate is not None else None, workspace.data_ptr(), plan.workspace_bytes,
               _cabi.status_word(device).data_ptr())
    return dy, dres, dpost, dpre, dgate


def gated_residual_norm(y: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                        pre_weight: torch.Tensor, gate: torch.Tensor | None = None,
                        residual_scale: float = 1.0, eps: float = 1e-6):
    """Returns ``(h, n)``: the new residual stream and the next block's normalised input.

    ``y`` and ``residual``: [..., D] of one type (fp16, bf16, fp32), D <= 16384.  ``post_weight``,
    ``pre_weight``: [D], and ``gate``: [D] (per channel), [..., 1] (per token) or [..., D] (per
    element), all of one type: that of ``y`` or fp32.  Gradients flow to every tensor argument;
    rows need not be contiguous with one another."""
    _cabi.refuse_tangents(y, residual, post_weight, pre_weight, gate)
    residual_scale, eps = _cabi.number("residual_scale", residual_scale), _cabi.number("eps", eps)
    key = (_cabi.signature(y, residual, post_weight, pre_weight, gate), residual_scale, eps)
    plan = _plans.get(key)
    if plan is None:
        plan = _cabi.remember(_plans, key, _NormPlan(y, residual, post_weight, pre_weight, gate, residual_scale, eps))
    if not plan.ready:  # as rows, and once more
        h, n = gated_residual_norm(*_as_rows(plan, y, residual, post_weight, pre_weight, gate), residual_scale, eps)
        return h.view(y.shape), n.view(y.shape)
    if torch.is_grad_enabled() and (y.requires_grad or residual.requires_grad or post_weight.requires_grad or
                                    pre_weight.requires_grad or (gate is not None and gate.requires_grad)):
        return _GatedResidualNorm.apply(y, residual, post_weight, pre_weight, gate, plan)
    h, n, _ = _forward(plan, y, residual, post_weight, pre_weight, gate, False)
    return h, n


def _as_rows(plan, y, residual, post_weight, pre_weight, gate):
    """The operands of a call whose plan is not ready, as the kernels take them."""
    if plan.form == _cabi.GATE_CHANNEL:
        gate = gate.contiguous()
    elif gate is not None:
        gate = _cabi.rows_view(gate.reshape(plan.shape[0], gate.shape[-1]))
    return (_cabi.rows_view(y.reshape(plan.shape)), _cabi.rows_view(residual.reshape(plan.shape)),
            post_weight.contiguous(), pre_weight.contiguous(), gate)


# The two passes as the custom operators call them: with operands of any strides and leading dimensions,
# the reciprocal norms kept between the passes in a tensor of their own.

def _ready_plan(y, residual, post_weight, pre_weight, gate, residual_scale, eps):
    operands = (y, residual, post_weight, pre_weight, gate)
    plan = _NormPlan(*operands, residual_scale, eps)
    if not plan.ready:
        operands = _as_rows(plan, *operands)
        plan = _NormPlan(*operands, residual_scale, eps)
    return plan, operands


def norm_forward_kept(y, residual, post_weight, pre_weight, gate, residual_scale, eps):
    plan, operands = _ready_plan(y, residual, post_weight, pre_weight, gate, residual_scale, eps)
    h, n, stats = _forward(plan, *operands, True)
    return h.view(y.shape), n.view(y.shape), stats


def norm_gradients_kept(dh, dn, y, residual, post_weight, pre_weight, gate, stats, residual_scale, eps):
    plan, operands = _ready_plan(y, residual, post_weight, pre_weight, gate, residual_scale, eps)
    dy, dres, dpost, dpre, dgate = _backward(plan, dh.reshape(plan.shape), dn.reshape(plan.shape), *operands, stats)
    return dy.view(y.shape), dres.view(y.shape), dpost, dpre, dgate if gate is None else dgate.view(gate.shape)


def _check(y, residual, post_weight, pre_weight, gate, eps) -> int:
    """Refuses what the kernels cannot take; returns the gate's form."""
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
    if rows > 1 << 30:
        raise ValueError("too many rows")
    return _gate_form(gate, rows, cols, lead)
