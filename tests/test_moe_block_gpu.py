"""Routing, the experts' products and the norms in a row, as a model runs them: values, gradients,
graphs, streams, and the torch custom ops."""
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwad

import tritonix_b200 as tnx
from oracle import moe as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
bf16, f32 = torch.bfloat16, torch.float32
NAMES = ("x", "residual", "logits", "w12", "w3", "post", "pre", "gate")


def make(t, n, d, f, seed=0, dtype=bf16):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": r(t, d).to(dtype), "residual": (2 * r(t, d)).to(dtype), "logits": r(t, n),
            "w12": (r(n, d, 2 * f) * d ** -0.5).to(dtype), "w3": (r(n, f, d) * f ** -0.5).to(dtype),
            "post": 1 + 0.1 * r(d), "pre": 1 + 0.1 * r(d), "gate": 0.5 + 0.1 * r(d), "bias": 0.1 * r(n),
            "dh": r(t, d).to(dtype), "dn": r(t, d).to(dtype)}


def leaves(case, grad=True):
    return [case[k].to(DEV).requires_grad_(grad) for k in NAMES]


KW = dict(scoring="sigmoid", num_groups=4, top_groups=2, scale=1.5, residual_scale=0.7)


def block(args, bias, top_k=3):
    x, residual, logits, w12, w3, post, pre, gate = args
    return tnx.moe_block(x, residual, logits, w12, w3, post, pre, top_k, bias=bias, gate=gate, **KW)


def reference(case, args):
    """The same from plain operations in 64 bits with autograd; experts as the oracle picks them."""
    x, residual, logits, w12, w3, post, pre, gate = args
    _, ids, _ = O.route_oracle(case["logits"], 3, "sigmoid", case["bias"], 4, 2)
    s = torch.sigmoid(logits).gather(1, ids)
    weights = 1.5 * s / s.sum(1, keepdim=True)
    y = torch.zeros_like(residual)
    for e in range(w12.shape[0]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        gu = x[token] @ w12[e]
        out = (torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]) @ w3[e]
        y = y.index_add(0, token, weights[token, slot].unsqueeze(1) * out)
    rms = lambda v: v * (v.square().mean(1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    h = 0.7 * residual + gate * rms(y) * post
    return h, rms(h) * pre


@pytest.mark.parametrize("t", [1, 7, 130, 900])
def test_block_and_its_gradients(t):
    case = make(t, 16, 256, 136, seed=t)
    args = leaves(case)
    h, n = block(args, case["bias"].to(DEV))
    grads = torch.autograd.grad([h, n], args, [case["dh"].to(DEV), case["dn"].to(DEV)])
    tnx.check_status(h.device)
    plain = [case[k].double().requires_grad_(True) for k in NAMES]
    rh, rn = reference(case, plain)
    want = torch.autograd.grad([rh, rn], plain, [case["dh"].double(), case["dn"].double()])
    # Values: the hidden activation, y and the result are rounded to bf16, half a step each.  On the
    # way back the gradient of y and that of the gate/up products are rounded too, and the backward
    # norm starts from the rounded y; each once, plus the result's own.  In the 2-norm independent
    # roundings of at most half a step stay below their sum.
    half = 2.0 ** -8
    for out, ref, roundings in ((h, rh, 3), (n, rn, 3)):
        assert (out.detach().cpu().double() - ref).norm() <= roundings * half * ref.norm()
    for grad, ref, name in zip(grads, want, NAMES):
        assert grad.shape == ref.shape
        assert (grad.cpu().double() - ref).norm() <= 6 * half * ref.norm(), name


def test_equals_the_three_operators():
    case = make(40, 16, 128, 64)
    args = leaves(case, False)
    h, n = block(args, case["bias"].to(DEV))
    w, i = tnx.route_experts(args[2], 3, scoring="sigmoid", bias=case["bias"].to(DEV), num_groups=4, top_groups=2,
                             scale=1.5)
    y = tnx.moe_swiglu(args[0], args[3], args[4], i, w)
    h2, n2 = tnx.gated_residual_norm(y, args[1], args[5], args[6], args[7], residual_scale=0.7)
    assert torch.equal(h, h2) and torch.equal(n, n2)


def test_training_step_captured_in_a_graph():
    case = make(200, 16, 256, 128, seed=5)
    args, bias = leaves(case), case["bias"].to(DEV)
    dh, dn = case["dh"].to(DEV), case["dn"].to(DEV)
    block(leaves(case, False), bias)     # warm-up on other leaves, without a graph of these
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, n = block(args, bias)
        grads = torch.autograd.grad([h, n], args, [dh, dn])
    other = make(200, 16, 256, 128, seed=6)
    with torch.no_grad():
        for a, k in zip(args, NAMES):
            a.copy_(other[k])
    graph.replay()
    fresh = leaves(other)
    h2, n2 = block(fresh, bias)
    want = torch.autograd.grad([h2, n2], fresh, [dh, dn])
    assert torch.equal(h, h2) and torch.equal(n, n2)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_two_streams_at_once():
    cases = [make(64, 16, 128, 64, seed=i) for i in (1, 2)]
    args = [leaves(c, False) for c in cases]
    bias = [c["bias"].to(DEV) for c in cases]
    want = [block(a, b) for a, b in zip(args, bias)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(8):
        for s, a, b in zip(streams, args, bias):
            with torch.cuda.stream(s):
                got.append(block(a, b))
    torch.cuda.synchronize()
    for i, (h, n) in enumerate(got):
        assert torch.equal(h, want[i % 2][0]) and torch.equal(n, want[i % 2][1])


def test_padding_tokens_leave_the_others_alone():
    """Rows of -inf logits and NaN inputs behind the last sequence."""
    case = make(50, 16, 128, 64, seed=9)
    clean = block(leaves(case, False), case["bias"].to(DEV))
    case["x"][40:] = float("nan")
    case["logits"][40:] = float("-inf")
    dirty = block(leaves(case, False), case["bias"].to(DEV))
    assert torch.equal(clean[0][:40], dirty[0][:40]) and torch.equal(clean[1][:40], dirty[1][:40])


def test_custom_ops():
    case = make(20, 16, 128, 64)
    args, bias = leaves(case, False), case["bias"].to(DEV)
    w, i = torch.ops.tritonix.route_experts(args[2], 3, "sigmoid", bias, 4, 2, True, 1.5)
    y = torch.ops.tritonix.moe_swiglu(args[0], args[3], args[4], i, w, "silu")
    h, n = torch.ops.tritonix.gated_residual_norm(y, args[1], args[5], args[6], args[7], 0.7, 1e-6)
    want = block(args, bias)
    assert torch.equal(h, want[0]) and torch.equal(n, want[1])


def test_forward_mode_differentiation_is_refused():
    """A tangent must not get lost, with gradients asked for and without, by itself or through a transform."""
    case = make(6, 16, 128, 64)
    args, bias = leaves(case, False), case["bias"].to(DEV)
    w, i = tnx.route_experts(args[2], 3)
    calls = ((args[2], lambda v: tnx.route_experts(v, 3)), (args[0], lambda v: tnx.moe_swiglu(v, args[3], args[4], i, w)),
             (w, lambda v: tnx.moe_swiglu(args[0], args[3], args[4], i, v)),
             *((args[j], lambda v, j=j: block(args[:j] + [v] + args[j + 1:], bias)) for j in range(8)))
    for value, call in calls:
        for grad in (False, True):
            with fwad.dual_level():
                dual = fwad.make_dual(value.clone().requires_grad_(grad), torch.ones_like(value))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(dual)
                call(value)  # (others are not disturbed by an open level)
        with pytest.raises(RuntimeError, match="forward-mode|storage"):  # (or torch's: a wrapped tensor has none)
            torch.func.jvp(call, (value,), (torch.ones_like(value),))


def block_of_ops(args, bias, top_k=3):
    x, residual, logits, w12, w3, post, pre, gate = args
    ops = torch.ops.tritonix
    w, i = ops.route_experts(logits, top_k, "sigmoid", bias, 4, 2, True, 1.5)
    return ops.gated_residual_norm(ops.moe_swiglu(x, w12, w3, i, w, "silu"), residual, post, pre, gate, 0.7, 1e-6)


@pytest.mark.parametrize("traced", [False, True])
def test_custom_ops_train(traced):
    """Through the custom operators, called and traced: the gradients of the Python functions."""
    case = make(60, 16, 256, 136, seed=8)
    bias, outs = case["bias"].to(DEV), [case["dh"].to(DEV), case["dn"].to(DEV)]
    args = leaves(case)
    want = block(args, bias)
    want_grads = torch.autograd.grad(want, args, outs)
    fn = torch.compile(block_of_ops, backend="aot_eager", fullgraph=True) if traced else block_of_ops
    args = leaves(case)
    with warnings.catch_warnings():
        warnings.filterwarnings("error", message=".*autograd kernel was not registered.*")
        got = fn(args, bias)
        grads = torch.autograd.grad(got, args, outs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(grads, want_grads))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(fn(args, bias), want))


def test_custom_ops_pass_torchs_own_checks():
    case = make(12, 16, 64, 32)
    x, residual, logits, w12, w3, post, pre, gate = leaves(case)
    w, i = tnx.route_experts(logits.detach(), 3)
    w.requires_grad_(True)
    ops = torch.ops.tritonix
    for op, args in ((ops.route_experts, (logits, 3, "softmax", None, 1, 1, False, 1.5)),
                     (ops.moe_swiglu, (x, w12, w3, i, w, "silu")),
                     (ops.moe_swiglu, (x.detach(), w12, w3.detach(), i.long(), w.detach(), "none")),
                     (ops.gated_residual_norm, (x, residual, post, pre, gate, 0.7, 1e-6)),
                     (ops.gated_residual_norm, (x, residual, post, pre, None, 0.7, 1e-6))):
        torch.library.opcheck(op.default, args)


def test_custom_ops_take_any_strides_and_leading_dimensions():
    case = make(24, 16, 64, 32, seed=3)
    x, residual, logits, w12, w3, post, pre, gate = leaves(case)
    out = [case["dh"].to(DEV), case["dn"].to(DEV)]
    ops = torch.ops.tritonix
    cols = lambda t: t.detach().mT.contiguous().mT.requires_grad_(True)  # noqa: E731
    w, i = tnx.route_experts(logits.detach(), 3)
    a = [x, w12, w3, w.requires_grad_(True)]
    b = [cols(x), cols(w12), cols(w3), cols(w)]
    grads = [torch.autograd.grad(ops.moe_swiglu(*v[:3], i, v[3], "silu"), v, out[0]) for v in (a, b)]
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    grads = [torch.autograd.grad(ops.route_experts(v, 3, "softmax", None, 1, 1, False, 1.0)[0], v, torch.ones_like(w))
             for v in (logits, cols(logits))]
    assert torch.equal(grads[0][0], grads[1][0])
    a, b = [x, residual, post, pre, gate], [t.detach().view(2, 12, 64).requires_grad_(True) for t in (x, residual)]
    ga = torch.autograd.grad(ops.gated_residual_norm(*a, 0.7, 1e-6), a, out)
    gb = torch.autograd.grad(ops.gated_residual_norm(*b, *a[2:], 0.7, 1e-6), b + a[2:], [t.view(2, 12, 64) for t in out])
    assert all(torch.equal(p, q.view(p.shape)) for p, q in zip(ga, gb))


def test_custom_ops_refuse_second_derivatives_and_tangents():
    case = make(6, 16, 64, 32)
    args = leaves(case)
    h, n = block_of_ops(args, case["bias"].to(DEV))
    with pytest.raises(RuntimeError, match="gradient of its own"):
        torch.autograd.grad(n.float().square().sum(), args, create_graph=True)
    for grad in (False, True):
        for j in range(8):
            with fwad.dual_level():
                dual = fwad.make_dual(args[j].detach().requires_grad_(grad), torch.ones_like(args[j]))
                others = [a.detach() for a in args]
                with pytest.raises(RuntimeError):
                    block_of_ops(others[:j] + [dual] + others[j + 1:], case["bias"].to(DEV))


@pytest.mark.parametrize("traced", [False, True])
def test_custom_ops_with_one_output_unused(traced):
    case = make(20, 16, 64, 32, seed=4)
    bias = case["bias"].to(DEV)
    for used in (0, 1):
        args = leaves(case)
        want = torch.autograd.grad(block(args, bias)[used].float().sum(), args, allow_unused=True)
        fn = lambda *a: block_of_ops(a, bias)[used]  # noqa: E731
        if traced:
            fn = torch.compile(fn, backend="aot_eager", fullgraph=True)
        args = leaves(case)
        got = torch.autograd.grad(fn(*args).float().sum(), args, allow_unused=True)
        for a, b in zip(want, got):
            assert torch.equal(a, b if b is not None else torch.zeros_like(a))
