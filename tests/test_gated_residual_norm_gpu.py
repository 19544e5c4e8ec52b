"""The gated residual norm and its gradients against the 64-bit oracle."""
import ctypes

import pytest
import torch

import tritonix_b200 as tnx
from oracle import moe as O
from tritonix_b200 import _cabi

pytestmark = pytest.mark.gpu
DEV = "cuda"
f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32

# fp32 arithmetic: a sum over a row is a tree of at most 16 + 10 additions, then a reciprocal root
# (2 ulp) and a handful of products, each 2^-24 relative to the terms' absolute values; the second
# norm sees the first one's error.  Gradients chain two more such sums.
FORWARD = 64 * 2.0 ** -24
BACKWARD = 192 * 2.0 ** -24


def within(out, ref, mag, fp32):
    half = torch.finfo(out.dtype).eps / 2
    out = out.cpu().double()
    tol = fp32 * mag * (1 + half) + half * ref.abs() + torch.finfo(f16).smallest_normal * 2 ** -11
    bad = (out - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, by up to {((out - ref).abs() / tol).max():.2f} x"


def make(t, d, dtype, wtype, gate, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    shape = {"none": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[gate]
    return {"y": r(t, d).to(dtype), "residual": (r(t, d) * scale).to(dtype), "post": (1 + 0.2 * r(d)).to(wtype),
            "pre": (1 + 0.2 * r(d)).to(wtype), "gate": None if shape is None else (0.5 + r(*shape)).to(wtype),
            "dh": r(t, d).to(dtype), "dn": r(t, d).to(dtype)}


def on_gpu(case, grad):
    names = ("y", "residual", "post", "pre", "gate")
    return [None if case[n] is None else case[n].to(DEV).requires_grad_(grad) for n in names]


def check(case, alpha=0.75, eps=1e-5, views=None):
    args = views or on_gpu(case, True)
    h, n = tnx.gated_residual_norm(*args, residual_scale=alpha, eps=eps)
    names = ("y", "residual", "post", "pre", "gate")
    ref = [case[k] for k in names]
    rh, rn, mh, mn = O.norm_oracle(*ref, alpha, eps)
    within(h.detach(), rh, mh, FORWARD)
    within(n.detach(), rn, mn, FORWARD)
    leaves = [a for a in args if a is not None]
    grads = torch.autograd.grad([h, n], leaves, [case["dh"].to(DEV), case["dn"].to(DEV)])
    want = O.norm_gradient_oracle(*ref, alpha, eps, case["dh"], case["dn"])
    rows = len(case["y"])
    for grad, leaf, name in zip(grads, leaves, names):
        assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
        # (column sums: each block adds its rows one after another, then 32 strands of blocks)
        fp32 = BACKWARD + (rows * 2.0 ** -24 if name in ("post", "pre", "gate") else 0)
        within(grad, *want[name], fp32)
    return h, n, grads


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype,wtype", [(bf16, bf16), (bf16, f32), (f16, f16), (f16, f32), (f32, f32)])
@pytest.mark.parametrize("t,d", [(1, 64), (5, 1), (3, 1000), (40, 4096), (7, 2051), (2, 8200)])
def test_forward_and_gradients(t, d, dtype, wtype, gate):
    if gate == "token" and d == 1:
        pytest.skip("a [rows, 1] gate over one column is the full form")
    check(make(t, d, dtype, wtype, gate, seed=d))


@pytest.mark.parametrize("d", [16384, 16383, 12296])
@pytest.mark.parametrize("dtype", [bf16, f32])
def test_longest_rows(d, dtype):
    check(make(3, d, dtype, dtype, "channel", seed=d))


@pytest.mark.parametrize("t", [147, 1000])
def test_many_rows(t):
    check(make(t, 256, bf16, f32, "channel", seed=t))
    check(make(t, 24, f32, f32, "token", seed=t))


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("t,d,dtype,wtype", [(595, 64, bf16, bf16), (1201, 2056, f16, f32), (700, 4096, bf16, f32),
                                             (601, 4100, f32, f32), (600, 8192, f16, f16), (613, 1001, f32, f32),
                                             (599, 2503, bf16, f32), (640, 5001, f32, f32), (592, 33, f16, f16)])
def test_rows_that_arrive_ahead(t, d, dtype, wtype, gate):
    """Enough rows for the kernels that walk them with copies a few rows ahead."""
    check(make(t, d, dtype, wtype, gate, seed=t))


@pytest.mark.parametrize("dtype,d", [(bf16, 16384), (f32, 16384), (bf16, 16383), (f16, 9001)])
def test_many_long_rows(dtype, d):
    check(make(597, d, dtype, dtype, "channel"))


def test_rows_that_arrive_ahead_from_an_odd_address():
    """The first row starts, and the last one ends, off a 16-byte boundary."""
    case = make(600, 301, bf16, bf16, "full", seed=8)
    args = on_gpu(case, False)
    want = tnx.gated_residual_norm(*args)
    views = []
    for i, name in enumerate(("y", "residual", "gate")):
        store = torch.empty(1 + i + 600 * 301, device=DEV, dtype=bf16)
        store[1 + i:].copy_(case[name].to(DEV).reshape(-1))
        views.append(store[1 + i:].view(600, 301))
    got = tnx.gated_residual_norm(views[0], views[1], args[2], args[3], views[2])
    # (rows moved by different amounts are read element by element, and their squares added in another
    # order: the last bit may differ)
    for a, b in zip(want, got):
        torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-6)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("dtype,wtype", [(bf16, bf16), (bf16, f32), (f32, f32)])
@pytest.mark.parametrize("t,d", [(601, 9), (605, 68), (1203, 1022), (777, 2051), (593, 4090), (594, 8185)])
def test_rows_that_start_between_boundaries(t, d, dtype, wtype, gate):
    """Every tensor's rows are moved alike: whole vectors, a partial one at either end."""
    check(make(t, d, dtype, wtype, gate, seed=t + d))


@pytest.mark.parametrize("dtype,wtype", [(bf16, f32), (f32, f32)])
def test_partial_vectors_leave_their_neighbours_alone(dtype, wtype):
    """Infinities and NaN right before and after a row of a wider tensor stay out of it."""
    case = make(640, 77, dtype, wtype, "full", seed=3)
    args = on_gpu(case, False)
    want = tnx.gated_residual_norm(*args)

    def inside(value, fill):  # rows 80 + 5 elements apart: moved as 77's are, to a vector of 8 or of 4
        store = torch.full((640, 85), fill, device=DEV, dtype=value.dtype)
        store[:, :77] = value
        return store[:, :77]

    got = tnx.gated_residual_norm(inside(args[0], float("nan")), inside(args[1], float("inf")), args[2], args[3],
                                  inside(args[4], float("-inf")))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_one_row_for_many():
    """Rows that repeat (a pitch of zero) or overlap, off the 16-byte boundaries and on them."""
    for d in (301, 304):
        case = make(700, d, bf16, bf16, "full", seed=9)
        args = on_gpu(case, False)
        store = torch.randn(3 * 699 + d, device=DEV).to(bf16)
        views = [args[0][:1].expand(700, d), store.as_strided((700, d), (3, 1)), args[2], args[3], args[4][:1].expand(700, d)]
        want = tnx.gated_residual_norm(*[v.contiguous() for v in views])
        got = tnx.gated_residual_norm(*views)
        for a, b in zip(want, got):   # (another order of a row's sum: the last bit may differ)
            torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-6)


def test_rows_apart():
    case = make(800, 520, bf16, bf16, "full", seed=4)
    padded = lambda t: torch.nn.functional.pad(t.to(DEV), (0, 24))[:, :520]  # noqa: E731
    args = on_gpu(case, False)
    want = tnx.gated_residual_norm(*args)
    got = tnx.gated_residual_norm(padded(case["y"]), padded(case["residual"]), args[2], args[3], padded(case["gate"]))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_inference_gives_the_same_values():
    case = make(9, 520, bf16, bf16, "channel")
    h, n, _ = check(case)
    with torch.no_grad():
        h2, n2 = tnx.gated_residual_norm(*on_gpu(case, False), residual_scale=0.75, eps=1e-5)
    assert torch.equal(h, h2) and torch.equal(n, n2)


def test_runs_are_bit_identical():
    case = make(700, 1024, bf16, f32, "channel")
    first, second = check(case)[2], check(case)[2]
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_zero_rows_and_zero_values():
    args = [torch.zeros(0, 16, device=DEV, requires_grad=True), torch.zeros(0, 16, device=DEV),
            torch.ones(16, device=DEV, requires_grad=True), torch.ones(16, device=DEV)]
    h, n = tnx.gated_residual_norm(*args)
    assert h.shape == n.shape == (0, 16)
    dy, dpost = torch.autograd.grad([h, n], [args[0], args[2]], [torch.zeros_like(h), torch.zeros_like(n)])
    assert dy.shape == (0, 16) and torch.equal(dpost, torch.zeros(16, device=DEV))
    case = make(4, 96, f32, f32, "channel")
    case["y"][1] = 0
    case["residual"][1] = 0
    check(case)


def test_views_and_leading_dimensions():
    case = make(12, 200, bf16, bf16, "full", seed=2)
    big = torch.zeros(12, 256, dtype=bf16, device=DEV)
    big[:, 13:213] = case["y"].to(DEV)                       # rows that start off a 16-byte boundary
    wide = torch.zeros(12, 456, dtype=bf16, device=DEV)
    wide[:, 256:] = case["residual"].to(DEV)
    args = on_gpu(case, False)
    ref = tnx.gated_residual_norm(*args)
    out = tnx.gated_residual_norm(big[:, 13:213], wide[:, 256:], *args[2:])
    # (another vector width adds a row's squares in another order: the last bit may differ)
    for a, b in zip(ref, out):
        torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-6)
    same = tnx.gated_residual_norm(args[0].view(3, 4, 200), args[1].view(3, 4, 200), args[2], args[3],
                                   args[4].view(3, 4, 200))
    assert all(torch.equal(a, b.view(12, 200)) for a, b in zip(ref, same))
    column = args[0].t().contiguous().t()                    # transposed storage
    assert all(torch.equal(a, b) for a, b in zip(ref, tnx.gated_residual_norm(column, *args[1:])))
    token = torch.full((1, 1), 0.5, device=DEV, dtype=bf16).expand(12, 1)  # broadcast gate
    gated = tnx.gated_residual_norm(*args[:4], token)
    assert torch.equal(gated[0], tnx.gated_residual_norm(*args[:4], token.contiguous())[0])


def test_broadcast_gradient_and_unused_output():
    case = make(6, 64, f32, f32, "channel")
    args = on_gpu(case, True)
    h, n = tnx.gated_residual_norm(*args)
    grads = torch.autograd.grad(n.sum(), args)   # dn is an expanded scalar, dh absent
    case["dn"], case["dh"] = torch.ones(6, 64), torch.zeros(6, 64)
    want = O.norm_gradient_oracle(*[case[k] for k in ("y", "residual", "post", "pre", "gate")], 1.0, 1e-6,
                                  case["dh"], case["dn"])
    for grad, name in zip(grads, ("y", "residual", "post", "pre", "gate")):
        within(grad, *want[name], BACKWARD)


def test_gradient_against_differences():
    case = make(3, 10, f32, f32, "channel", seed=5)
    args = on_gpu(case, True)
    h, n = tnx.gated_residual_norm(*args, residual_scale=0.5, eps=1e-3)
    grads = torch.autograd.grad([h, n], args, [case["dh"].to(DEV), case["dn"].to(DEV)])
    names = ("y", "residual", "post", "pre", "gate")

    def value(which, delta):
        vals = [case[k].double() + (delta if k == which else 0) for k in names]
        hh, nn, _, _ = O.norm_oracle(*vals, 0.5, 1e-3)
        return (hh * case["dh"].double()).sum() + (nn * case["dn"].double()).sum()

    for grad, name in zip(grads, names):
        flat = case[name].double().reshape(-1)
        for i in range(0, flat.numel(), 3):
            delta = torch.zeros_like(flat)
            delta[i] = 1e-4
            delta = delta.view(case[name].shape)
            diff = (value(name, delta) - value(name, -delta)) / 2e-4
            # the step's square times a third derivative of a few tens, and fp32 in the gradient
            assert abs(grad.reshape(-1)[i].item() - diff.item()) <= 1e-5 * (1 + abs(diff.item()))


def test_captured_forward_and_backward():
    case = make(33, 512, bf16, f32, "channel")
    args = on_gpu(case, True)
    dh, dn = case["dh"].to(DEV), case["dn"].to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # warm-up; its graph is released before the capture
        h, n = tnx.gated_residual_norm(*args)
        torch.autograd.grad([h, n], args, [dh, dn])
        del h, n
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, n = tnx.gated_residual_norm(*args)
        grads = torch.autograd.grad([h, n], args, [dh, dn])
    with torch.no_grad():
        args[0].copy_(torch.randn(33, 512))
    graph.replay()
    fresh = [a.detach().clone().requires_grad_(True) for a in args]
    h2, n2 = tnx.gated_residual_norm(*fresh)
    want = torch.autograd.grad([h2, n2], fresh, [dh, dn])
    assert torch.equal(h, h2) and torch.equal(n, n2)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_offsets_past_32_bits():
    """140000 rows of 16384: 2.3e9 elements."""
    t, d = 140000, 16384
    case = make(40, d, bf16, bf16, "channel", seed=1)
    y, residual = torch.zeros(t, d, device=DEV, dtype=bf16), torch.zeros(t, d, device=DEV, dtype=bf16)
    for part, name in ((y, "y"), (residual, "residual")):
        part[:20].copy_(case[name][:20])
        part[-20:].copy_(case[name][20:])
    h, n = tnx.gated_residual_norm(y, residual, *[case[k].to(DEV) for k in ("post", "pre", "gate")], residual_scale=0.75)
    tnx.check_status(h.device)
    rh, rn, mh, mn = O.norm_oracle(*[case[k] for k in ("y", "residual", "post", "pre", "gate")], 0.75, 1e-6)
    within(torch.cat([h[:20], h[-20:]]), rh, mh, FORWARD)
    within(torch.cat([n[:20], n[-20:]]), rn, mn, FORWARD)
    assert not h[20:-20:997].any()


def test_refusals():
    y = torch.zeros(4, 8, device=DEV, dtype=bf16)
    w = torch.ones(8, device=DEV, dtype=bf16)
    fine = dict(y=y, residual=y, post_weight=w, pre_weight=w)
    for bad, match in (({"residual": y[:3]}, "shape"), ({"residual": y.float()}, "share"),
                       ({"post_weight": w[:7]}, "post_weight"), ({"pre_weight": w.float()}, "share one type"),
                       ({"gate": torch.ones(4, device=DEV, dtype=bf16)}, "gate must be"),
                       ({"gate": w.float()}, "share one type"), ({"eps": 0.0}, "eps"), ({"eps": float("nan")}, "eps"),
                       ({"post_weight": w.half(), "pre_weight": w.half()}, "share one type")):
        with pytest.raises(ValueError, match=match):
            tnx.gated_residual_norm(**{**fine, **bad})
    long = torch.zeros(1, 16385, device=DEV)
    with pytest.raises(ValueError, match="16384"):
        tnx.gated_residual_norm(long, long, long[0], long[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        tnx.gated_residual_norm(y.cpu(), y, w, w)


def test_a_scale_held_in_a_tensor_is_read_by_every_call():
    case = make(5, 96, f32, f32, "none")
    args, scale, eps = on_gpu(case, False), torch.tensor(1.0), torch.tensor(1e-6)
    for value in (1.0, 2.0, -0.5):
        scale.fill_(value)
        eps.fill_(abs(value) * 1e-3)
        want = tnx.gated_residual_norm(*args, residual_scale=value, eps=eps.item())
        got = tnx.gated_residual_norm(*args, residual_scale=scale, eps=eps)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(ValueError, match="residual_scale"):
        tnx.gated_residual_norm(*args, residual_scale=scale.requires_grad_(True))


@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("dtype,wtype", [(bf16, bf16), (f16, f32), (f32, f32)])
@pytest.mark.parametrize("t,d", [(594, 1), (600, 2), (601, 3), (598, 5), (1203, 7), (700, 8)])
def test_many_rows_shorter_than_a_copy(t, d, dtype, wtype, gate):
    """Several rows share the 16 bytes at either end of a tensor."""
    check(make(t, d, dtype, wtype, gate, seed=t + d))


@pytest.mark.parametrize("dtype,d", [(bf16, 3), (bf16, 301), (f32, 2), (f32, 77)])
def test_first_and_last_rows_between_boundaries(dtype, d):
    """Tensors that start and end anywhere, NaN and infinities right before and behind them."""
    case = make(640, d, dtype, dtype, "full", seed=d)
    args = on_gpu(case, False)
    want = tnx.gated_residual_norm(*args)
    for at in range(1, 16 // case["y"].element_size()):
        views = []
        for value, name in zip((float("nan"), float("inf"), float("-inf")), ("y", "residual", "gate")):
            store = torch.full((at + 640 * d + 9,), value, device=DEV, dtype=dtype)
            store[at:at + 640 * d] = case[name].to(DEV).reshape(-1)
            views.append(store[at:at + 640 * d].view(640, d))
        got = tnx.gated_residual_norm(views[0], views[1], args[2], args[3], views[2])
        # (another order of a row's sum: the last bit may differ)
        for a, b in zip(want, got):
            torch.testing.assert_close(a.float(), b.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)


@pytest.mark.parametrize("pitch", [0, 3, 8])
@pytest.mark.parametrize("d", [301, 304])
def test_c_entry_points_take_rows_that_overlap(d, pitch):
    """The Python function copies such rows first; the C functions read them as they lie."""
    rows = 700
    case = make(rows, d, bf16, f32, "full", seed=d)
    _, residual, post, pre, gate = on_gpu(case, False)
    store = torch.randn(pitch * (rows - 1) + d, generator=torch.Generator().manual_seed(pitch)).to(bf16)
    case["y"] = store.as_strided((rows, d), (pitch, 1)).contiguous()
    y = store.to(DEV)
    dh, dn = case["dh"].to(DEV), case["dn"].to(DEV)
    problem = _cabi.NormProblem(rows, d, _cabi.BF16, _cabi.F32, _cabi.GATE_FULL, 0.75, 1e-5, 0, pitch, d, d)
    h, n, dy, dres = (torch.full((rows, d), float("nan"), device=DEV, dtype=bf16) for _ in range(4))
    dgate = torch.full((rows, d), float("nan"), device=DEV)
    dpost, dpre = torch.empty(d, device=DEV), torch.empty(d, device=DEV)
    stats = torch.empty(rows, 2, device=DEV)
    status = _cabi.status_word(y.device).data_ptr()
    size = _cabi.lib.tnx_gated_residual_norm_workspace(ctypes.byref(problem))
    workspace = torch.empty(size, device=DEV, dtype=torch.uint8)
    at = lambda *tensors: [t.data_ptr() for t in tensors]  # noqa: E731
    _cabi.call(y.device, _cabi.lib.tnx_gated_residual_norm, ctypes.byref(problem),
               *at(y, residual, post, pre, gate, h, n, stats), status)
    _cabi.call(y.device, _cabi.lib.tnx_gated_residual_norm_backward, ctypes.byref(problem), dh.data_ptr(), d,
               dn.data_ptr(), d, *at(y, residual, post, pre, gate, stats, dy, dres, dpost, dpre, dgate, workspace), size,
               status)
    ref = [case[k] for k in ("y", "residual", "post", "pre", "gate")]
    rh, rn, mh, mn = O.norm_oracle(*ref, 0.75, 1e-5)
    within(h, rh, mh, FORWARD)
    within(n, rn, mn, FORWARD)
    want = O.norm_gradient_oracle(*ref, 0.75, 1e-5, case["dh"], case["dn"])
    for grad, name in ((dy, "y"), (dres, "residual"), (dpost, "post"), (dpre, "pre"), (dgate, "gate")):
        within(grad, *want[name], BACKWARD + (rows * 2.0 ** -24 if name in ("post", "pre") else 0))
