"""What the C entry points of routing and the norm refuse, without a device."""
import ctypes

import pytest
import torch

import tritonix_b200 as tnx
from tritonix_b200 import _cabi

lib = _cabi.lib
PTR = 1 << 20  # never dereferenced: every call here is refused before a launch


def route(**kw):
    p = _cabi.RouteProblem(tokens=4, experts=64, top_k=4, groups=1, top_groups=1, scoring=0, renormalize=1,
                           dtype=_cabi.F32, scale=1.0, stride_logits=64)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(experts=0), dict(experts=513), dict(top_k=0), dict(top_k=33),
                                 dict(experts=8, top_k=9), dict(groups=0), dict(groups=5), dict(groups=64, top_groups=4),
                                 dict(groups=8, top_groups=0), dict(groups=8, top_groups=9),
                                 dict(groups=32, top_groups=1), dict(scoring=2), dict(dtype=3), dict(stride_logits=-1)])
def test_route_refuses(bad):
    p = route(**bad)
    assert lib.tnx_route_experts(ctypes.byref(p), PTR, None, PTR, PTR, None) == _cabi.ERR_INVALID
    assert lib.tnx_route_experts_backward(ctypes.byref(p), PTR, PTR, PTR, PTR, None) == _cabi.ERR_INVALID
    assert _cabi.last_error()


def test_route_null_and_empty():
    assert lib.tnx_route_experts(None, PTR, None, PTR, PTR, None) == _cabi.ERR_INVALID
    assert lib.tnx_route_experts(ctypes.byref(route()), None, None, PTR, PTR, None) == _cabi.ERR_INVALID
    assert lib.tnx_route_experts_backward(ctypes.byref(route()), PTR, None, PTR, PTR, None) == _cabi.ERR_INVALID
    assert lib.tnx_route_experts(ctypes.byref(route(tokens=0)), None, None, None, None, None) == _cabi.OK


def norm(**kw):
    p = _cabi.NormProblem(rows=4, cols=64, dtype=_cabi.BF16, weight_dtype=_cabi.BF16, gate_form=0,
                          residual_scale=1.0, eps=1e-6, stride_y=64, stride_residual=64, stride_gate=64)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


def forward(p, y=PTR, gate=PTR):
    return lib.tnx_gated_residual_norm(ctypes.byref(p), y, PTR, PTR, PTR, gate, PTR, PTR, None, None, None)


def backward(p, workspace=PTR, nbytes=1 << 30, stats=PTR, dgate=PTR):
    return lib.tnx_gated_residual_norm_backward(ctypes.byref(p), PTR, 64, PTR, 64, PTR, PTR, PTR, PTR, PTR, stats, PTR,
                                                PTR, PTR, PTR, dgate, workspace, nbytes, None, None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=0), dict(cols=16385), dict(dtype=4), dict(weight_dtype=_cabi.F16),
                                 dict(gate_form=4), dict(eps=0.0), dict(eps=float("nan")), dict(stride_y=-64)])
def test_norm_refuses(bad):
    assert forward(norm(**bad)) == _cabi.ERR_INVALID
    assert backward(norm(**bad)) == _cabi.ERR_INVALID


def test_norm_null_and_workspace():
    assert forward(norm(), y=None) == _cabi.ERR_INVALID
    assert forward(norm(gate_form=1), gate=None) == _cabi.ERR_INVALID
    assert backward(norm(), stats=None) == _cabi.ERR_INVALID
    assert backward(norm(gate_form=2), dgate=None) == _cabi.ERR_INVALID
    need = lib.tnx_gated_residual_norm_workspace(ctypes.byref(norm()))
    assert need == 4 * 2 * 64 * 4
    assert lib.tnx_gated_residual_norm_workspace(ctypes.byref(norm(gate_form=1))) == 4 * 3 * 64 * 4
    assert backward(norm(), nbytes=need - 1) == _cabi.ERR_INVALID
    assert backward(norm(), workspace=PTR + 4) == _cabi.ERR_INVALID
    assert forward(norm(rows=0), y=None) == _cabi.OK


def moe(**kw):
    p = _cabi.MoeProblem(tokens=10, experts=4, top_k=2, d_model=64, d_ff=32, n_out=48, dtype=_cabi.BF16,
                         activation=_cabi.EPI_GLU_SILU, wide_ids=0, train=0, stride_x=64, stride_w12e=64 * 64,
                         stride_w12k=64, stride_w3e=32 * 48, stride_w3k=48, stride_y=48)
    for key, value in kw.items():
        setattr(p, key, value)
    return p


def query(p):
    res = _cabi.MoeResources()
    return lib.tnx_moe_query(ctypes.byref(p), ctypes.byref(res)), res


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(experts=0), dict(experts=513), dict(top_k=0), dict(d_model=60),
                                 dict(d_ff=0), dict(n_out=4), dict(dtype=_cabi.F32), dict(activation=0),
                                 dict(activation=4), dict(tokens=1 << 28, top_k=2), dict(stride_x=56), dict(stride_x=68),
                                 dict(stride_w12k=56), dict(stride_w12e=64 * 64 - 8), dict(stride_w3e=0),
                                 dict(stride_w12k=0), dict(stride_y=40), dict(d_model=1 << 21, stride_x=1 << 21),
                                 dict(tokens=1 << 27, n_out=1 << 20, stride_y=1 << 20, stride_w3k=1 << 20,
                                      stride_w3e=1 << 25)])
def test_moe_refuses(bad):
    p = moe(**bad)
    assert query(p)[0] == _cabi.ERR_INVALID and _cabi.last_error()
    assert lib.tnx_moe_swiglu(ctypes.byref(p), PTR, PTR, PTR, PTR, PTR, PTR, None, PTR, 1 << 40, None,
                              None) == _cabi.ERR_INVALID


def test_moe_resources_and_workspace():
    rc, res = query(moe())
    # 20 pairs on 4 experts: a tile for each expert, rows padded to multiples of 16
    assert rc == _cabi.OK and (res.tile_rows, res.max_tiles) == (256, 4)
    rows = 20 + 4 * 15
    part = rows * 48 * 4
    assert res.workspace_bytes >= part + rows * 32 * 2
    rc, train = query(moe(train=1))
    assert rc == _cabi.OK and train.workspace_bytes >= part and train.saved_bytes >= rows * 32 * 10
    assert query(moe(tokens=4000))[1].max_tiles == 4 + (8000 - 4) // 256

    def forward(p, nbytes, workspace=PTR, saved=None, x=PTR):
        return lib.tnx_moe_swiglu(ctypes.byref(p), x, PTR, PTR, PTR, PTR, PTR, saved, workspace, nbytes, None, None)

    assert forward(moe(), res.workspace_bytes - 1) == _cabi.ERR_INVALID
    assert forward(moe(), res.workspace_bytes, workspace=PTR + 16) == _cabi.ERR_INVALID
    assert forward(moe(), res.workspace_bytes, x=None) == _cabi.ERR_INVALID
    assert forward(moe(), res.workspace_bytes, x=PTR + 2) == _cabi.ERR_INVALID
    assert forward(moe(train=1), 1 << 30) == _cabi.ERR_INVALID                     # nothing to save into
    assert forward(moe(tokens=0), 0, workspace=None, x=None) == _cabi.OK

    def gradients(p, nbytes, dy=PTR, stride=48, workspace=PTR, saved=PTR):
        return lib.tnx_moe_swiglu_backward(ctypes.byref(p), dy, stride, PTR, PTR, PTR, saved, PTR, PTR, PTR, PTR,
                                           workspace, nbytes, None, None)

    need = train.backward_workspace_bytes
    for kw in (dict(nbytes=need - 1), dict(nbytes=need, workspace=PTR + 128), dict(nbytes=need, saved=PTR + 128),
               dict(nbytes=need, saved=None), dict(nbytes=need, dy=None), dict(nbytes=need, stride=44),
               dict(nbytes=need, stride=40), dict(nbytes=need, dy=PTR + 8)):
        assert gradients(moe(train=1), **kw) == _cabi.ERR_INVALID


def test_custom_ops_give_shapes_without_a_device():
    meta = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="meta")  # noqa: E731
    w, i = torch.ops.tritonix.route_experts(meta(5, 8), 2, "softmax", None, 1, 1, True, 1.0)
    assert (w.shape, w.dtype, i.shape, i.dtype) == ((5, 2), torch.float32, (5, 2), torch.int32)
    y = torch.ops.tritonix.moe_swiglu(meta(5, 16), meta(8, 16, 48), meta(8, 24, 32), i, w, "silu")
    assert (y.shape, y.dtype) == ((5, 32), torch.bfloat16)
    h, n = torch.ops.tritonix.gated_residual_norm(y, y, meta(32), meta(32), None, 1.0, 1e-6)
    assert h.shape == n.shape == (5, 32)


def test_host_tensors_are_refused():
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        tnx.route_experts(x, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        tnx.gated_residual_norm(x, x, x[0], x[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        tnx.moe_swiglu(x, torch.zeros(2, 8, 16), torch.zeros(2, 8, 8), torch.zeros(4, 1, dtype=torch.int32),
                       torch.zeros(4, 1))


@pytest.mark.parametrize("n,d,f,n_out,match", [(4, 60, 32, 48, "multiples of 8"), (4, 64, 30, 48, "multiples of 8"),
                                               (4, 64, 32, 60, "multiples of 8"), (4, 0, 32, 48, "multiples of 8"),
                                               (4, 64, 0, 48, "multiples of 8"), (4, 64, 32, 0, "multiples of 8"),
                                               (4, 4, 32, 48, "multiples of 8"), (0, 64, 32, 48, "experts"),
                                               (513, 64, 32, 48, "experts")])
@pytest.mark.parametrize("t", [0, 1, 4])
def test_sizes_that_no_copy_could_mend_are_refused(monkeypatch, t, n, d, f, n_out, match):
    """Contiguous operands of sizes that the products do not take: refused before any of them is copied."""
    monkeypatch.setattr(_cabi, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(torch.Tensor, "clone", None)
    half = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match=match):
        tnx.moe_swiglu(half(t, d), half(n, d, 2 * f), half(n, f, n_out), torch.zeros(t, 2, dtype=torch.int32),
                       torch.zeros(t, 2))


@pytest.mark.parametrize("dtype,wdtype", [(_cabi.BF16, _cabi.BF16), (_cabi.F16, _cabi.F32), (_cabi.F32, _cabi.F32)])
@pytest.mark.parametrize("rows", [592, 593, 594, 598, 601, 1203])
@pytest.mark.parametrize("gate_form", [0, 3])
def test_bulk_copies_stay_inside_their_tensors(gate_form, rows, dtype, wdtype):
    """Rows from one element on, pitches from the row's own length on, tensors that start anywhere."""
    size, wsize = (4 if dtype == _cabi.F32 else 2), (4 if wdtype == _cabi.F32 else 2)
    copied = set()
    for cols in (*range(1, 40), 63, 64, 301, 2049, 4096):
        for apart in (0, 1, 3, 8):
            for at in range(0, 16, 2):
                p = norm(rows=rows, cols=cols, dtype=dtype, weight_dtype=wdtype, gate_form=gate_form,
                         stride_y=cols + apart, stride_residual=cols, stride_gate=cols + apart)
                base = (PTR + at // size * size, PTR + (at + 6) // size * size, PTR + at // wsize * wsize)
                n = lib.tnx_selftest_norm_copies(ctypes.byref(p), *base)
                assert n in (0, -1), (cols, apart, at, n)
                if n == 0:
                    copied.add(cols)
    assert {64, 301, 2049} <= copied
    assert lib.tnx_selftest_norm_copies(ctypes.byref(norm(rows=rows, cols=0)), PTR, PTR, PTR) == -2
    assert lib.tnx_selftest_norm_copies(ctypes.byref(norm(rows=500, cols=64)), PTR, PTR, PTR) == -1


@pytest.mark.parametrize("pitch", [0, 8])
def test_bulk_copies_of_one_row_for_many(pitch):
    p = norm(rows=700, cols=304, stride_y=pitch, stride_residual=304)
    assert lib.tnx_selftest_norm_copies(ctypes.byref(p), PTR, PTR, None) == 0
    assert lib.tnx_selftest_norm_copies(ctypes.byref(p), PTR + 2, PTR, None) == -1


def test_custom_ops_carry_gradients_without_a_device():
    """Traced with tensors that hold no data, outputs ask for gradients and their shapes come back."""
    meta = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="meta", requires_grad=True)  # noqa: E731
    ops = torch.ops.tritonix
    logits, x, w12, w3 = meta(5, 8, dt=torch.float32), meta(5, 16), meta(8, 16, 48), meta(8, 24, 32)
    res, post, pre, gate = meta(5, 32), meta(32, dt=torch.float32), meta(32, dt=torch.float32), meta(5, 1, dt=torch.float32)
    w, i = ops.route_experts(logits, 2, "softmax", None, 1, 1, True, 1.0)
    assert w.requires_grad and not i.requires_grad
    y = ops.moe_swiglu(x, w12, w3, i, w, "silu")
    h, n = ops.gated_residual_norm(y, res, post, pre, gate, 1.0, 1e-6)
    leaves = [logits, x, w12, w3, res, post, pre, gate]
    grads = torch.autograd.grad([h, n], leaves, [torch.empty_like(h), torch.empty_like(n)])
    assert [(g.shape, g.dtype) for g in grads] == [(v.shape, v.dtype) for v in leaves]
    # one leaf alone, none at all
    y = ops.moe_swiglu(x.detach(), w12, w3.detach(), i, w.detach(), "silu")
    assert torch.autograd.grad(y, w12, torch.empty_like(y))[0].shape == w12.shape
    assert not ops.moe_swiglu(x.detach(), w12.detach(), w3.detach(), i, w.detach(), "silu").requires_grad
    with torch.no_grad():
        assert not ops.moe_swiglu(x, w12, w3, i, w, "silu").requires_grad
    with torch.inference_mode():
        assert ops.moe_swiglu(x, w12, w3, i, w, "silu").shape == (5, 32)


@pytest.mark.parametrize("tokens", [2 ** 31 - 3, 2 ** 31 - 1])
def test_route_refuses_more_tokens_than_it_can_number(tokens):
    assert lib.tnx_route_experts(ctypes.byref(route(tokens=tokens)), PTR, None, PTR, PTR, None) == _cabi.ERR_INVALID
    assert "tokens" in _cabi.last_error()
