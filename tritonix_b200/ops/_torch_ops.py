"""Registers the contraction kernels as torch custom operators (namespace ``tritonix``) so
they are visible to ``torch.ops``, autograd-free tracing and ``torch.compile`` (fake kernels
give the output shapes).  The mixture-of-experts operators have gradients here too: where one is
asked for, the operator becomes ``<name>_train``, which also returns what ``<name>_backward``
needs, so that a traced training step holds both passes.  ``cfg`` is the tnx_config of include/tritonix_b200.h as a list of
ints in field order (tile_m, tile_n, tile_k, stages, acc_stages, cta_group, split_k, group_m,
tile_order, kernel, max_ctas); missing trailing entries and zeros select the defaults.
"""
from __future__ import annotations

from typing import List

import torch

from tritonix_b200 import _cabi

_FIELDS = ("tile_m", "tile_n", "tile_k", "stages", "acc_stages", "cta_group", "split_k",
           "group_m", "tile_order", "kernel", "max_ctas")

_lib = torch.library.Library("tritonix", "DEF")
_lib.define("gemm(Tensor a, Tensor b, int[] cfg) -> Tensor")
_lib.define("gemm_splitk(Tensor a, Tensor b, int split_k, int[] cfg) -> Tensor")
_lib.define("glu(Tensor x, Tensor w12, int activation, int[] cfg) -> Tensor")
_lib.define("conv2d_forward(Tensor input, Tensor weight, Tensor? bias, int[] stride, int[] padding, "
            "int[] dilation, int[] cfg) -> Tensor")
# (scoring and activation by name, as the Python functions take them)
_lib.define("route_experts(Tensor logits, int top_k, str scoring, Tensor? bias, int num_groups, int top_groups, "
            "bool renormalize, float scale) -> (Tensor, Tensor)")
_lib.define("moe_swiglu(Tensor x, Tensor w12, Tensor w3, Tensor ids, Tensor weights, str activation) -> Tensor")
_lib.define("gated_residual_norm(Tensor y, Tensor residual, Tensor post_weight, Tensor pre_weight, Tensor? gate, "
            "float residual_scale, float eps) -> (Tensor, Tensor)")
# (gradients: empty tensors where none is wanted)
_lib.define("route_experts_train(Tensor logits, int top_k, str scoring, Tensor? bias, int num_groups, int top_groups, "
            "bool renormalize, float scale) -> (Tensor, Tensor)")
_lib.define("route_experts_backward(Tensor dweights, Tensor logits, Tensor ids, str scoring, bool renormalize, "
            "float scale) -> Tensor")
_lib.define("moe_swiglu_train(Tensor x, Tensor w12, Tensor w3, Tensor ids, Tensor weights, str activation) "
            "-> (Tensor, Tensor)")
_lib.define("moe_swiglu_backward(Tensor dy, Tensor x, Tensor w12, Tensor w3, Tensor ids, Tensor saved, str activation, "
            "bool[4] wants) -> (Tensor, Tensor, Tensor, Tensor)")
_lib.define("gated_residual_norm_train(Tensor y, Tensor residual, Tensor post_weight, Tensor pre_weight, Tensor? gate, "
            "float residual_scale, float eps) -> (Tensor, Tensor, Tensor)")
_lib.define("gated_residual_norm_backward(Tensor dh, Tensor dn, Tensor y, Tensor residual, Tensor post_weight, "
            "Tensor pre_weight, Tensor? gate, Tensor stats, float residual_scale, float eps) "
            "-> (Tensor, Tensor, Tensor, Tensor, Tensor)")


def cfg_to_list(cfg: dict | None) -> List[int]:
    c = _cabi.make_config(cfg)
    return [int(getattr(c, f)) for f in _FIELDS]


def _cfg_dict(cfg: List[int]) -> dict:
    return {f: int(v) for f, v in zip(_FIELDS, cfg) if int(v) != 0}


def _gemm(a, b, cfg):
    c = torch.empty((a.shape[0], b.shape[1]), device=a.device, dtype=a.dtype)
    _cabi.launch(a, b, c, _cfg_dict(cfg))
    return c


def _gemm_splitk(a, b, split_k, cfg):
    c = torch.empty((a.shape[0], b.shape[1]), device=a.device, dtype=a.dtype)
    _cabi.launch(a, b, c, {**_cfg_dict(cfg), "split_k": int(split_k)})
    return c


def _glu(x, w12, activation, cfg):
    z = torch.empty((x.shape[0], w12.shape[1] // 2), device=x.device, dtype=x.dtype)
    _cabi.launch(x, w12, z, _cfg_dict(cfg), epilogue=int(activation))
    return z


def _conv_out_shape(input, weight, stride, padding, dilation):
    n, _, h, w = input.shape
    c_out, _, r, s = weight.shape
    h_out = (h + 2 * padding[0] - dilation[0] * (r - 1) - 1) // stride[0] + 1
    w_out = (w + 2 * padding[1] - dilation[1] * (s - 1) - 1) // stride[1] + 1
    return (n, c_out, h_out, w_out)


def _conv2d_forward(input, weight, bias, stride, padding, dilation, cfg):
    from tritonix_b200.ops.conv2d import conv2d_forward
    config = _cfg_dict(cfg)
    return conv2d_forward(input, weight, bias, tuple(stride), tuple(padding), tuple(dilation),
                          config=config or None)


def _route_experts(logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale):
    from tritonix_b200.ops.moe import route_experts
    return route_experts(logits, top_k, scoring=scoring, bias=bias, num_groups=num_groups, top_groups=top_groups,
                         renormalize=renormalize, scale=scale)


def _moe_swiglu(x, w12, w3, ids, weights, activation):
    from tritonix_b200.ops.moe import moe_swiglu
    return moe_swiglu(x, w12, w3, ids, weights, activation)


def _gated_residual_norm(y, residual, post_weight, pre_weight, gate, residual_scale, eps):
    from tritonix_b200.ops.norm import gated_residual_norm
    return gated_residual_norm(y, residual, post_weight, pre_weight, gate, residual_scale, eps)


_lib.impl("route_experts", _route_experts, "CUDA")
_lib.impl("moe_swiglu", _moe_swiglu, "CUDA")
_lib.impl("gated_residual_norm", _gated_residual_norm, "CUDA")
_lib.impl("gemm", _gemm, "CUDA")
_lib.impl("conv2d_forward", _conv2d_forward, "CUDA")
_lib.impl("gemm_splitk", _gemm_splitk, "CUDA")
_lib.impl("glu", _glu, "CUDA")


@torch.library.register_fake("tritonix::gemm")
def _gemm_fake(a, b, cfg):
    return a.new_empty((a.shape[0], b.shape[1]))


@torch.library.register_fake("tritonix::gemm_splitk")
def _gemm_splitk_fake(a, b, split_k, cfg):
    return a.new_empty((a.shape[0], b.shape[1]))


@torch.library.register_fake("tritonix::glu")
def _glu_fake(x, w12, activation, cfg):
    return x.new_empty((x.shape[0], w12.shape[1] // 2))


@torch.library.register_fake("tritonix::conv2d_forward")
def _conv2d_forward_fake(input, weight, bias, stride, padding, dilation, cfg):
    channels_last = (not input.is_contiguous()
                     and input.is_contiguous(memory_format=torch.channels_last))
    return torch.empty(_conv_out_shape(input, weight, stride, padding, dilation),
                       device=input.device, dtype=input.dtype,
                       memory_format=torch.channels_last if channels_last
                       else torch.contiguous_format)


@torch.library.register_fake("tritonix::route_experts")
def _route_experts_fake(logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale):
    shape = (logits.shape[0], top_k)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.register_fake("tritonix::moe_swiglu")
def _moe_swiglu_fake(x, w12, w3, ids, weights, activation):
    return x.new_empty((x.shape[0], w3.shape[2]))


@torch.library.register_fake("tritonix::gated_residual_norm")
def _gated_residual_norm_fake(y, residual, post_weight, pre_weight, gate, residual_scale, eps):
    return y.new_empty(y.shape), y.new_empty(y.shape)


# ------------------------------------------------------------------- gradients of the operators above

def _asks_for_gradient(args) -> bool:
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args)


def _with_training_form(name: str, outputs: int) -> None:
    """Autograd's entry of operator ``name``: its training form where a gradient is asked for."""
    plain, train = getattr(torch.ops.tritonix, name).default, getattr(torch.ops.tritonix, name + "_train").default

    def call(*args):
        if _asks_for_gradient(args):
            out = train(*args)
            return out[0] if outputs == 1 else out[:outputs]
        with torch._C._AutoDispatchBelowAutograd():
            return plain(*args)

    _lib.impl(name, call, "Autograd")


def _once_differentiable(name: str) -> None:
    backward = getattr(torch.ops.tritonix, name).default

    def call(*args):
        if _asks_for_gradient(args):
            raise RuntimeError(f"tritonix::{name} has no gradient of its own")
        with torch._C._AutoDispatchBelowAutograd():
            return backward(*args)

    _lib.impl(name, call, "Autograd")


def _route_experts_train(logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale):
    with torch.no_grad():
        return _route_experts(logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale)


def _route_experts_backward(dweights, logits, ids, scoring, renormalize, scale):
    from tritonix_b200.ops.moe import route_gradient
    return route_gradient(dweights, logits, ids, scoring, renormalize, scale)


def _moe_swiglu_train(x, w12, w3, ids, weights, activation):
    from tritonix_b200.ops.moe import moe_forward_kept
    return moe_forward_kept(x, w12, w3, ids, weights, activation)


def _moe_swiglu_backward(dy, x, w12, w3, ids, saved, activation, wants):
    from tritonix_b200.ops.moe import moe_gradients_kept
    grads = moe_gradients_kept(dy, x, w12, w3, ids, saved, activation, wants)
    return tuple(x.new_empty(0) if g is None else g for g in grads)


def _gated_residual_norm_train(y, residual, post_weight, pre_weight, gate, residual_scale, eps):
    from tritonix_b200.ops.norm import norm_forward_kept
    return norm_forward_kept(y, residual, post_weight, pre_weight, gate, residual_scale, eps)


def _gated_residual_norm_backward(dh, dn, y, residual, post_weight, pre_weight, gate, stats, residual_scale, eps):
    from tritonix_b200.ops.norm import norm_gradients_kept
    *grads, dgate = norm_gradients_kept(dh, dn, y, residual, post_weight, pre_weight, gate, stats, residual_scale, eps)
    return (*grads, y.new_empty(0) if dgate is None else dgate)


for _name, _fn in (("route_experts_train", _route_experts_train), ("route_experts_backward", _route_experts_backward),
                   ("moe_swiglu_train", _moe_swiglu_train), ("moe_swiglu_backward", _moe_swiglu_backward),
                   ("gated_residual_norm_train", _gated_residual_norm_train),
                   ("gated_residual_norm_backward", _gated_residual_norm_backward)):
    _lib.impl(_name, _fn, "CUDA")

torch.library.register_fake("tritonix::route_experts_train", _route_experts_fake)


@torch.library.register_fake("tritonix::route_experts_backward")
def _route_experts_backward_fake(dweights, logits, ids, scoring, renormalize, scale):
    return logits.new_empty(logits.shape)


@torch.library.register_fake("tritonix::moe_swiglu_train")
def _moe_swiglu_train_fake(x, w12, w3, ids, weights, activation):
    from tritonix_b200.ops.moe import moe_saved_bytes
    return x.new_empty((x.shape[0], w3.shape[2])), \
        x.new_empty(moe_saved_bytes(x, w12, w3, ids, activation), dtype=torch.uint8)


@torch.library.register_fake("tritonix::moe_swiglu_backward")
def _moe_swiglu_backward_fake(dy, x, w12, w3, ids, saved, activation, wants):
    shapes = ((x.shape, x.dtype), (w12.shape, x.dtype), (w3.shape, x.dtype), (ids.shape, torch.float32))
    return tuple(x.new_empty(shape, dtype=dtype) if want else x.new_empty(0)
                 for (shape, dtype), want in zip(shapes, wants))


@torch.library.register_fake("tritonix::gated_residual_norm_train")
def _gated_residual_norm_train_fake(y, residual, post_weight, pre_weight, gate, residual_scale, eps):
    return y.new_empty(y.shape), y.new_empty(y.shape), \
        y.new_empty((y.numel() // y.shape[-1], 2), dtype=torch.float32)


@torch.library.register_fake("tritonix::gated_residual_norm_backward")
def _gated_residual_norm_backward_fake(dh, dn, y, residual, post_weight, pre_weight, gate, stats, residual_scale, eps):
    return y.new_empty(y.shape), y.new_empty(y.shape), post_weight.new_empty(post_weight.shape), \
        post_weight.new_empty(post_weight.shape), y.new_empty(0) if gate is None else gate.new_empty(gate.shape)


def _route_experts_context(ctx, inputs, output):
    logits, _, ctx.scoring, _, _, _, ctx.renormalize, ctx.scale = inputs
    ctx.save_for_backward(logits, output[1])


def _route_experts_vjp(ctx, dweights, _):
    logits, ids = ctx.saved_tensors
    grad = torch.ops.tritonix.route_experts_backward(dweights, logits, ids, ctx.scoring, ctx.renormalize, ctx.scale)
    return grad, None, None, None, None, None, None, None


def _moe_swiglu_context(ctx, inputs, output):
    *operands, _, ctx.activation = inputs
    ctx.save_for_backward(*operands, output[1])


def _moe_swiglu_vjp(ctx, dy, _):
    x, w12, w3, ids, saved = ctx.saved_tensors
    needs = ctx.needs_input_grad
    wants = [needs[0], needs[1], needs[2], needs[4]]
    grads = torch.ops.tritonix.moe_swiglu_backward(dy, x, w12, w3, ids, saved, ctx.activation, wants)
    dx, dw12, dw3, dweights = (g if want else None for g, want in zip(grads, wants))
    return dx, dw12, dw3, None, dweights, None


def _gated_residual_norm_context(ctx, inputs, output):
    *operands, ctx.residual_scale, ctx.eps = inputs
    ctx.save_for_backward(*operands, output[2])


def _gated_residual_norm_vjp(ctx, dh, dn, _):
    *operands, gate, stats = ctx.saved_tensors
    *grads, dgate = torch.ops.tritonix.gated_residual_norm_backward(dh, dn, *operands, gate, stats, ctx.residual_scale,
                                                                    ctx.eps)
    return (*grads, None if gate is None else dgate, None, None)


for _name, _outputs, _vjp, _context in (("route_experts", 2, _route_experts_vjp, _route_experts_context),
                                        ("moe_swiglu", 1, _moe_swiglu_vjp, _moe_swiglu_context),
                                        ("gated_residual_norm", 2, _gated_residual_norm_vjp,
                                         _gated_residual_norm_context)):
    torch.library.register_autograd(f"tritonix::{_name}_train", _vjp, setup_context=_context, lib=_lib)
    _with_training_form(_name, _outputs)
    _once_differentiable(_name + "_backward")
