"""Experts' gated products and their gradients against the 64-bit oracle."""
import ctypes

import pytest
import torch

import tritonix_b200 as tnx
from oracle import moe as O
from tritonix_b200 import _cabi

pytestmark = pytest.mark.gpu
DEV = "cuda"
f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32


def make(t, n, k, d, f, n_out, dtype, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if ids is None:
        ids = r(t, n).topk(k, dim=1).indices.to(torch.int32)
    return {"x": r(t, d).to(dtype), "w12": (r(n, d, 2 * f) * d ** -0.5).to(dtype),
            "w3": (r(n, f, n_out) * f ** -0.5).to(dtype), "weights": torch.softmax(r(t, k), 1), "ids": ids,
            "dy": r(t, n_out).to(dtype)}


def operands(case, grad=False):
    return [case[name].to(DEV).requires_grad_(grad and name != "ids") for name in ("x", "w12", "w3", "ids", "weights")]


def close(out, ref, roundings, name):
    """Norm of the difference: `roundings` independent ones to the operands' type between the inputs
    and the result, each of at most half a step relative to a value (together at most their sum),
    and fp32 sums of a few thousand terms.  Per element: the same against the result's size, with
    room for the largest of many."""
    out, half = out.detach().cpu().double(), torch.finfo(out.dtype).eps / 2 if out.dtype != f32 else 0.0
    assert out.shape == ref.shape and torch.isfinite(out).all(), name
    norm = ref.norm()
    bound = roundings + 2e-6
    assert (out - ref).norm() <= bound * norm + 1e-30, f"{name}: {(out - ref).norm() / norm:.2e} > {bound:.2e}"
    if norm > 0:
        rms = ref.square().mean().sqrt()
        worst = ((out - ref).abs() / (ref.abs() + rms)).max()
        assert worst <= 8 * bound + half, f"{name}: an element is {worst:.2e} off"


def check(case, activation="silu", train=True):
    half = torch.finfo(case["x"].dtype).eps / 2
    cpu = [case[n] for n in ("x", "w12", "w3", "ids", "weights")]
    args = operands(case)
    y = tnx.moe_swiglu(*args, activation=activation)
    tnx.check_status(y.device)
    want = O.experts_oracle(*cpu, activation, case["dy"] if train else None)
    # rounded twice: the hidden activation and the result
    close(y, want[0] if train else want, 2 * half, "y")
    if not train:
        return
    leaves = operands(case, True)
    y2 = tnx.moe_swiglu(*leaves, activation=activation)
    assert y2.dtype == y.dtype
    close(y2, want[0], 2 * half, "y (training)")
    x, w12, w3, _, weights = leaves
    grads = torch.autograd.grad(y2, [x, w12, w3, weights], case["dy"].to(DEV))
    tnx.check_status(y.device)
    # the gradient of the gate/up products is rounded, and the result; dw3 meets the hidden
    # activation's rounding instead; the routing weights' gradient is fp32 throughout
    # (exp and the division in the gate: 2^-21 each)
    for grad, ref, name in zip(grads, want[1:], ("dx", "dw12", "dw3", "dweights")):
        close(grad, ref, 2 * half if name != "dweights" else 2.0 ** -20, name)
    return grads


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("t,n,k,d,f,n_out", [(1, 4, 2, 64, 64, 64), (1, 1, 1, 8, 8, 8), (5, 8, 2, 72, 40, 24),
                                             (37, 3, 3, 200, 136, 264), (130, 16, 4, 256, 128, 256),
                                             (300, 4, 1, 328, 200, 520), (33, 60, 6, 136, 264, 128)])
def test_single_cta_tiles(t, n, k, d, f, n_out, dtype):
    check(make(t, n, k, d, f, n_out, dtype, seed=t + d))


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("t,n,k,d,f,n_out", [(800, 2, 1, 136, 200, 264), (1000, 4, 2, 256, 128, 256),
                                             (700, 1, 1, 64, 320, 72)])
def test_cta_pairs(t, n, k, d, f, n_out, dtype):
    check(make(t, n, k, d, f, n_out, dtype, seed=t + d))


@pytest.mark.parametrize("activation", ["silu", "sigmoid", "none"])
def test_activations(activation):
    check(make(50, 4, 2, 128, 96, 64, bf16), activation)
    check(make(1, 4, 2, 128, 96, 64, bf16), activation, train=False)


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("n,k,d,f,n_out", [(64, 8, 512, 264, 2056), (16, 8, 1032, 136, 72), (2, 1, 4104, 1048, 16),
                                           (4, 8, 72, 40, 24), (300, 32, 64, 64, 64), (40, 33, 64, 64, 64)])
def test_one_token(n, k, d, f, n_out, dtype):
    ids = None if k <= n else torch.randint(0, n, (1, k), generator=torch.Generator().manual_seed(n))
    check(make(1, n, k, d, f, n_out, dtype, seed=n, ids=ids), train=False)


@pytest.mark.parametrize("ids", [[3, 3, 3], [-1, 5, 3], [0, 6, 2 ** 31 - 1], [-1, -1, -1]])
def test_one_token_with_ids_out_of_range_and_repeated(ids):
    for wide in (torch.int32, torch.int64):
        case = make(1, 6, 3, 136, 72, 40, bf16, ids=torch.tensor([ids], dtype=wide))
        check(case, train=False)
        if max(ids) < 0:
            assert not tnx.moe_swiglu(*operands(case)).any()


def test_many_pairs_use_the_chunked_plan():
    check(make(3001, 24, 3, 64, 40, 48, bf16, seed=9))
    check(make(2100, 7, 4, 32, 24, 40, f16, seed=4))


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_ids_out_of_range_and_repeated(wide):
    t, n, k = 90, 6, 3
    ids = torch.randint(0, n, (t, k), generator=torch.Generator().manual_seed(1))
    ids[::4, 0] = -1
    ids[1::5, 1] = n
    ids[7] = -1                      # a token no expert takes
    ids[8] = 2                       # the same expert three times
    ids[9] = 2 ** 31 - 1
    if wide == torch.int64:
        ids[10] = 2 ** 32            # would be expert 0 in 32 bits
        ids[11] = -2 ** 40
    case = make(t, n, k, 96, 64, 72, bf16, ids=ids.to(wide))
    grads = check(case)
    assert torch.equal(grads[0][7].cpu(), torch.zeros(96, dtype=bf16))
    assert not grads[3].cpu()[(case["ids"] < 0) | (case["ids"] >= n)].any()
    none = make(5, n, k, 96, 64, 72, bf16, ids=torch.full((5, k), -1, dtype=wide))
    x, w12, w3, i, w = operands(none, True)
    y = tnx.moe_swiglu(x, w12, w3, i, w)
    assert torch.equal(y, torch.zeros_like(y))
    for g in torch.autograd.grad(y, [x, w12, w3, w], none["dy"].to(DEV)):
        assert torch.equal(g, torch.zeros_like(g))


def test_one_expert_takes_all_and_others_get_zero_gradients():
    ids = torch.zeros(400, 1, dtype=torch.int32) + 3
    grads = check(make(400, 5, 1, 72, 64, 136, bf16, ids=ids))
    for e in (0, 1, 2, 4):
        assert not grads[1][e].any() and not grads[2][e].any()


def test_no_tokens():
    case = make(0, 4, 2, 64, 64, 64, bf16, ids=torch.empty(0, 2, dtype=torch.int32))
    x, w12, w3, ids, w = operands(case, True)
    y = tnx.moe_swiglu(x, w12, w3, ids, w)
    assert y.shape == (0, 64)
    dx, dw12, dw3, dw = torch.autograd.grad(y, [x, w12, w3, w], case["dy"].to(DEV))
    assert dx.shape == (0, 64) and dw.shape == (0, 2) and not dw12.any() and not dw3.any()


def test_nan_and_inf_rows_stay_their_own():
    case = make(60, 4, 2, 64, 64, 64, bf16)
    clean = tnx.moe_swiglu(*operands(case))
    case["x"][13] = float("nan")
    case["x"][21] = float("inf")
    dirty = tnx.moe_swiglu(*operands(case))
    keep = [i for i in range(60) if i not in (13, 21)]
    assert torch.equal(clean[keep], dirty[keep])
    assert torch.isnan(dirty[13]).all() and not torch.isfinite(dirty[21]).any()


def test_strided_operands():
    case = make(40, 4, 2, 64, 64, 72, bf16)
    x, w12, w3, ids, w = operands(case)
    want = tnx.moe_swiglu(x, w12, w3, ids, w)
    pad = lambda t, n: torch.nn.functional.pad(t, (0, n))[..., :t.shape[-1]]  # noqa: E731
    wide = lambda t: torch.stack((t, torch.full_like(t, float("nan"))), 1)[:, 0]  # noqa: E731
    # padded rows, matrices apart, columns stored first, an odd pitch, transposed ids
    for args in ((pad(x, 8), pad(w12, 16), pad(w3, 8), ids, w), (x, wide(w12), wide(w3), ids, w),
                 (x.t().contiguous().t(), w12.mT.contiguous().mT, w3, ids.t().contiguous().t(), w),
                 (pad(x, 3), pad(w12, 1), w3, ids, w.t().contiguous().t())):
        assert torch.equal(tnx.moe_swiglu(*args), want)
    shared = tnx.moe_swiglu(x, w12[:1].expand(4, -1, -1), w3[:1].expand(4, -1, -1), ids, w)
    assert torch.equal(shared, tnx.moe_swiglu(x, w12[:1].repeat(4, 1, 1), w3[:1].repeat(4, 1, 1), ids, w))


def test_gradients_of_some_operands_only_and_runs_are_bit_identical():
    case = make(260, 8, 2, 128, 72, 136, bf16)
    want = check(case)
    dy = case["dy"].to(DEV)
    for i, name in enumerate(("x", "w12", "w3", "weights")):
        args = operands(case)
        leaf = args[i if i < 3 else 4].requires_grad_(True)
        (grad,) = torch.autograd.grad(tnx.moe_swiglu(*args), leaf, dy)
        assert torch.equal(grad, want[i]), name
    # a broadcast gradient
    x, *rest = operands(case)
    x.requires_grad_(True)
    (a,) = torch.autograd.grad(tnx.moe_swiglu(x, *rest).sum(), x)
    (b,) = torch.autograd.grad(tnx.moe_swiglu(x, *rest), x, torch.ones_like(dy))
    assert torch.equal(a, b)


def test_weights_gradient_against_differences():
    case = make(6, 3, 2, 32, 24, 16, f16)
    *args, w = operands(case)
    w.requires_grad_(True)
    (grad,) = torch.autograd.grad(tnx.moe_swiglu(*args, w), w, case["dy"].to(DEV))
    cpu = [case[n] for n in ("x", "w12", "w3", "ids")]
    for t in range(6):
        for s in range(2):
            delta = torch.zeros(6, 2, dtype=torch.float64)
            delta[t, s] = 0.5   # the output is linear in the weights: any step will do
            up = O.experts_oracle(*cpu, case["weights"].double() + delta)
            down = O.experts_oracle(*cpu, case["weights"].double() - delta)
            diff = ((up - down) * case["dy"].double()).sum().item()
            assert abs(grad[t, s].item() - diff) <= 1e-5 * (1 + abs(diff))


def test_other_stream_and_captured_graphs_do_not_share_scratch():
    a, b = make(70, 8, 2, 128, 64, 64, bf16, seed=1), make(70, 8, 2, 128, 64, 64, bf16, seed=2)
    want = [tnx.moe_swiglu(*operands(c)) for c in (a, b)]
    args = [operands(c) for c in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s, arg in zip(streams, args):
            with torch.cuda.stream(s):
                outs.append(tnx.moe_swiglu(*arg))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))
    graphs, held = [], []
    for arg in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(tnx.moe_swiglu(*arg))
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(h, w) for h, w in zip(held, want))
        for h in held:
            h.zero_()
    # the routing of a replayed graph is the one in its buffers now
    args[0][3].copy_(args[1][3])
    graphs[0].replay()
    assert torch.equal(held[0], tnx.moe_swiglu(*args[0]))


def test_captured_backward():
    case = make(200, 8, 2, 128, 64, 72, bf16)
    want = check(case)
    leaves = operands(case, True)
    dy = case["dy"].to(DEV)
    inputs = [leaves[i] for i in (0, 1, 2, 4)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(tnx.moe_swiglu(*leaves), inputs, dy)
    for g in grads:
        g.zero_()
    graph.replay()
    assert all(torch.equal(g, w) for g, w in zip(grads, want))


def test_offsets_past_32_bits():
    """320000 rows x 8192 fp32 sums between the down product and the join: 2.6e9 elements."""
    t, n, k, d, f, n_out = 40000, 8, 8, 64, 64, 8192
    case = make(64, n, k, d, f, n_out, bf16, seed=2)
    g = torch.Generator().manual_seed(3)
    ids = torch.stack([torch.randperm(n, generator=g)[:k] for _ in range(t)]).to(torch.int32)
    x = torch.randn(t, d, generator=g).to(bf16)
    weights = torch.rand(t, k, generator=g)
    y = tnx.moe_swiglu(x.to(DEV), case["w12"].to(DEV), case["w3"].to(DEV), ids.to(DEV), weights.to(DEV))
    tnx.check_status(y.device)
    pick = torch.cat([torch.arange(20), torch.randint(0, t, (40,), generator=g), torch.arange(t - 20, t)])
    want = O.experts_oracle(x[pick], case["w12"], case["w3"], ids[pick], weights[pick])
    close(y[pick.to(DEV)], want, 2 * torch.finfo(bf16).eps / 2, "y")


def test_refusals():
    x, w12, w3, ids, w = operands(make(4, 4, 2, 64, 64, 64, bf16))
    for bad, match in (((x.float(), w12, w3, ids, w), "float16"), ((x, w12.half(), w3, ids, w), "float16"),
                       ((x[0], w12, w3, ids, w), "expects"), ((x[:, :32], w12, w3, ids, w), "fit"),
                       ((x, w12[:3], w3, ids, w), "fit"), ((x, w12, w3[:, :32], ids, w), "fit"),
                       ((x, w12, w3, ids[:3], w), "ids"), ((x, w12, w3, ids.float(), w), "ids"),
                       ((x, w12, w3, ids[:, :0], w[:, :0]), "ids"), ((x, w12, w3, ids, w[:, :1]), "weights"),
                       ((x, w12, w3, ids, w.double()), "weights"), ((x, w12, w3[:, :, :60], ids, w), "multiples of 8"),
                       ((x[:, :60], w12[:, :60], w3, ids, w), "multiples of 8")):
        with pytest.raises(ValueError, match=match):
            tnx.moe_swiglu(*bad)
    with pytest.raises(ValueError, match="activation"):
        tnx.moe_swiglu(x, w12, w3, ids, w, activation="relu")
    with pytest.raises(ValueError, match="512"):
        tnx.moe_swiglu(x, w12[:1].expand(513, -1, -1), w3[:1].expand(513, -1, -1), ids, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        tnx.moe_swiglu(x.cpu(), w12, w3, ids, w)


@pytest.mark.parametrize("d,f,n_out", [(60, 32, 48), (64, 30, 48), (64, 32, 60)])
def test_contiguous_operands_of_odd_sizes_are_refused(d, f, n_out):
    with pytest.raises(ValueError, match="multiples of 8"):
        tnx.moe_swiglu(*operands(make(4, 4, 2, d, f, n_out, bf16)))


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("t,d,f,n_out", [(500, 4096, 136, 2048), (340, 2056, 72, 4104), (270, 2048, 264, 2048)])
def test_long_sums_that_feed_the_routing_weights_gradient(t, d, f, n_out, dtype):
    """Sums over thousands of elements in many parts, for more rows of an expert than a warp holds in
    registers at once.  An accumulator that ran over all of K would be short by 3e-9 K of its size
    (6e-6 at K = 2048) in each of the gradient's factors, past the bound of 2.95e-6."""
    ids = (torch.arange(t) % 2).to(torch.int32).unsqueeze(1)
    check(make(t, 2, 1, d, f, n_out, dtype, seed=d, ids=ids))


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("t,n,k,d,f,n_out", [(5, 2, 1, 264, 2048, 256), (40, 3, 2, 64, 1160, 72), (2, 4, 2, 128, 4104, 264)])
def test_down_products_in_slices(t, n, k, d, f, n_out, dtype):
    """Few tiles and a long K: slices of it (the last one short) are added by the join."""
    case = make(t, n, k, d, f, n_out, dtype, seed=f)
    problem = _cabi.MoeProblem(t, n, k, d, f, n_out, _cabi.DTYPES[dtype], _cabi.EPI_GLU_SILU, 0, 1, d, d * 2 * f, 2 * f,
                               f * n_out, n_out, n_out)
    res = _cabi.MoeResources()
    assert _cabi.lib.tnx_moe_query(ctypes.byref(problem), ctypes.byref(res)) == _cabi.OK
    rows = t * k // 16 * 16   # (at least; a copy of the rows of x and one of the fp32 rows per slice)
    assert res.workspace_bytes >= (t * k + min(n, t * k) * 15) // 16 * 16 * (2 * d + 2 * 4 * n_out) > rows * 4 * n_out
    check(case)


@pytest.mark.parametrize("t", [1, 70])
def test_small_weights_in_fp16(t):
    """The hidden activation is rounded with its weight: where that leaves fp16's normal range, to
    half its smallest step (2^-25) instead of half a step of the value."""
    case = make(t, 4, 2, 128, 96, 64, f16, seed=t)
    case["weights"] = 10.0 ** -torch.linspace(1, 7, 2 * t).view(t, 2)
    y = tnx.moe_swiglu(*operands(case)).cpu().double()
    ref, tol = O.experts_oracle(*[case[n] for n in ("x", "w12", "w3", "ids", "weights")]), torch.zeros(t, 64).double()
    half, step = 2.0 ** -11, 2.0 ** -25
    x, w12, w3 = (case[n].double() for n in ("x", "w12", "w3"))
    for e in range(4):
        token, slot = torch.nonzero(case["ids"] == e, as_tuple=True)
        gu = x[token] @ w12[e]
        hidden = case["weights"][token, slot].double().unsqueeze(1) * torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]
        # (and 2^-18 for sums of 128 and 96 terms in fp32, the exponential and the division)
        tol.index_add_(0, token, ((half + 2.0 ** -18) * hidden.abs() + step) @ w3[e].abs())
    tol += half * ref.abs() + step
    assert ((y - ref).abs() <= tol).all()
