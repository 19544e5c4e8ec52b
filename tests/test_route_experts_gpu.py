"""Routing to experts against the 64-bit oracle: the same experts in the same order, weights and
gradients to fp32 accuracy."""
import pytest
import torch

import tritonix_b200 as tnx
from oracle import moe as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32

# fp32 scores: expf (2 ulp), a division and a sum of up to 512 terms by a tree of depth 21, each
# rounding 2^-24 relative, twice when renormalised; 40 roundings cover the chain
WEIGHT_RTOL = 40 * 2.0 ** -24


def make(t, n, dtype, seed, bias):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(t, n, generator=g) * 1.5).to(dtype)
    return logits, (torch.randn(n, generator=g) * 0.1 if bias else None), g


def check(logits, k, g=None, **kw):
    bias = kw.pop("bias", None)
    oracle = dict(scoring=kw.get("scoring", "softmax"), groups=kw.get("num_groups", 1),
                  top_groups=kw.get("top_groups", 1), renormalize=kw.get("renormalize", True),
                  scale=kw.get("scale", 1.0))
    weights, ids = tnx.route_experts(logits.to(DEV), k, bias=None if bias is None else bias.to(DEV), **kw)
    assert weights.dtype == f32 and ids.dtype == torch.int32 and weights.shape == ids.shape == (len(logits), k)
    w, i, _ = O.route_oracle(logits, k, bias=bias, **oracle)
    assert torch.equal(ids.cpu().long(), i)
    torch.testing.assert_close(weights.cpu().double(), w, rtol=WEIGHT_RTOL, atol=1e-37)
    return weights, ids


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("t,n,k", [(1, 8, 2), (3, 1, 1), (37, 33, 7), (130, 64, 6), (64, 256, 8), (9, 512, 32)])
def test_plain(t, n, k, bias, scoring, dtype):
    logits, b, _ = make(t, n, dtype, t + n + k, bias)
    check(logits, k, bias=b, scoring=scoring, scale=2.5)
    check(logits, k, bias=b, scoring=scoring, renormalize=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("t,n,k,groups,top", [(50, 256, 8, 8, 4), (33, 60, 5, 3, 2), (20, 32, 3, 32, 5),
                                              (21, 160, 6, 20, 3), (7, 24, 8, 4, 4), (5, 34, 17, 2, 1)])
def test_groups(t, n, k, groups, top, bias, scoring):
    logits, b, _ = make(t, n, f32, n + groups, bias)
    check(logits, k, bias=b, scoring=scoring, num_groups=groups, top_groups=top)


@pytest.mark.parametrize("dtype", [bf16, f32])
def test_ties_go_to_the_lowest_index(dtype):
    logits = torch.zeros(6, 96).to(dtype)
    logits[1, 40:] = 1.0
    logits[2, ::2] = -1.0
    logits[3] = torch.arange(96) // 4
    logits[4, 5] = -0.0
    for kw in ({}, {"bias": torch.full((96,), 0.25)}, {"num_groups": 8, "top_groups": 3}):
        check(logits, 10, **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top", [(1, 1), (8, 3)])
def test_choices_closer_than_fp32_can_tell(scoring, groups, top):
    """A bias that makes all choices equal up to its own rounding: only 64 bits tell them apart."""
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        logits = torch.randn(1, 128, generator=g) * 2
        s = torch.softmax(logits.double(), 1) if scoring == "softmax" else torch.sigmoid(logits.double())
        check(logits, 8, bias=(0.75 - s[0]).float(), scoring=scoring, num_groups=groups, top_groups=top)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_infinities_and_nan(scoring):
    inf, nan = float("inf"), float("nan")
    logits = torch.randn(6, 40, generator=torch.Generator().manual_seed(3))
    logits[0] = -inf                       # nothing left
    logits[1, 3:] = -inf                   # fewer finite than picks
    logits[2, ::2] = -inf
    logits[3] = torch.finfo(f32).min
    logits[4, 7] = 1e4                     # everything else underflows
    check(logits, 5, scoring=scoring)
    check(logits, 5, scoring=scoring, renormalize=False)
    check(logits, 5, scoring=scoring, num_groups=4, top_groups=2)
    logits[5, 11] = nan
    weights, ids = tnx.route_experts(logits[:, :30].to(DEV), 30, scoring=scoring)
    assert torch.equal(ids.cpu().long().sort(1).values, torch.arange(30).expand(6, 30))
    assert ids[5, -1].item() == 11
    assert torch.equal(weights[0].cpu(), torch.zeros(30))
    # bias and groups: still distinct and in range
    _, ids = tnx.route_experts(logits.to(DEV), 20, scoring=scoring, num_groups=4, top_groups=2,
                               bias=torch.zeros(40, device=DEV))
    assert all(len(set(r)) == 20 and 0 <= min(r) and max(r) < 40 for r in ids.cpu().tolist())


def test_strides_and_empty():
    g = torch.Generator().manual_seed(1)
    big = torch.randn(40, 200, generator=g)
    ref, ids = check(big[:, 3:67].contiguous(), 4)
    for view in (big.to(DEV)[:, 3:67], big.t().contiguous().to(DEV).t()[:, 3:67]):
        w, i = tnx.route_experts(view, 4)
        assert torch.equal(w, ref) and torch.equal(i, ids)
    w, i = tnx.route_experts(torch.empty(0, 8, device=DEV), 2)
    assert w.shape == i.shape == (0, 2)
    w, i = tnx.route_experts(torch.randn(8, device=DEV).expand(5, 8), 2)
    assert torch.equal(i, i[:1].expand(5, 2))


@pytest.mark.parametrize("dtype", [f16, bf16, f32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("t,n,k,groups,top", [(1, 8, 2, 1, 1), (70, 64, 6, 1, 1), (33, 200, 8, 4, 2), (11, 512, 32, 1, 1)])
def test_gradient(t, n, k, groups, top, renormalize, scoring, dtype):
    logits, bias, g = make(t, n, dtype, n + k, True)
    dw = torch.randn(t, k, generator=g)
    leaf = logits.to(DEV).requires_grad_(True)
    weights, ids = tnx.route_experts(leaf, k, scoring=scoring, bias=bias.to(DEV), num_groups=groups,
                                     top_groups=top, renormalize=renormalize, scale=1.5)
    assert not ids.requires_grad
    (grad,) = torch.autograd.grad(weights, leaf, dw.to(DEV))
    assert grad.dtype == dtype
    ref = O.route_gradient_oracle(logits, ids.cpu().long(), dw, scoring, renormalize, 1.5)
    # the terms that cancel are of the size of s (|dw| + sum |dw| s); one rounding to the type
    scores = torch.softmax(logits.double(), 1) if scoring == "softmax" else torch.sigmoid(logits.double())
    if renormalize:
        scores = scores / scores.gather(1, ids.cpu().long()).sum(1, keepdim=True)
    size = 1.5 * scores.clamp(max=1) * 2 * dw.abs().double().sum(1, keepdim=True)
    tol = 64 * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).smallest_normal * 2 ** -9
    assert ((grad.cpu().double() - ref).abs() <= tol).all()


def test_gradient_against_differences():
    logits, bias, g = make(5, 12, f32, 7, True)
    dw = torch.randn(5, 3, generator=g)
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            leaf = logits.to(DEV).requires_grad_(True)
            w, ids = tnx.route_experts(leaf, 3, scoring=scoring, bias=bias.to(DEV), renormalize=renormalize)
            (grad,) = torch.autograd.grad(w, leaf, dw.to(DEV))
            step, z = 1e-4, logits.double()
            for e in range(12):
                delta = torch.zeros_like(z)
                delta[:, e] = step

                def value(v):
                    s = torch.softmax(v, 1) if scoring == "softmax" else torch.sigmoid(v)
                    p = s.gather(1, ids.cpu().long())
                    return ((p / p.sum(1, keepdim=True) if renormalize else p) * dw.double()).sum(1)

                diff = (value(z + delta) - value(z - delta)) / (2 * step)
                # central differences: step^2 / 6 times a third derivative of a few |dw|
                torch.testing.assert_close(grad[:, e].cpu().double(), diff, rtol=0, atol=1e-6)


def test_captured_and_replayed():
    logits = torch.randn(64, 64, device=DEV)
    bias = torch.zeros(64, device=DEV)
    tnx.route_experts(logits, 4, bias=bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, i = tnx.route_experts(logits, 4, bias=bias)
    for seed in range(3):
        logits.copy_(torch.randn(64, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        w2, i2 = tnx.route_experts(logits, 4, bias=bias)
        assert torch.equal(w, w2) and torch.equal(i, i2)


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    for kw, match in (({"top_k": 0}, "top_k"), ({"top_k": 9}, "top_k"), ({"num_groups": 3}, "groups"),
                      ({"num_groups": 4, "top_groups": 1, "top_k": 3}, "top_k"),
                      ({"num_groups": 4, "top_groups": 5}, "groups"), ({"scoring": "relu"}, "scoring")):
        with pytest.raises(ValueError, match=match):
            tnx.route_experts(x, **{"top_k": 2, **kw})
    with pytest.raises(ValueError, match="bias"):
        tnx.route_experts(x, 2, bias=torch.zeros(7, device=DEV))
    with pytest.raises(ValueError, match="bias"):
        tnx.route_experts(x, 2, bias=torch.zeros(8, device=DEV, dtype=bf16))
    with pytest.raises(ValueError, match="2-D"):
        tnx.route_experts(x[0], 2)
    with pytest.raises(ValueError, match="2-D"):
        tnx.route_experts(x.long(), 2)
    with pytest.raises(ValueError, match="512"):
        tnx.route_experts(torch.zeros(1, 513, device=DEV), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        tnx.route_experts(x.cpu(), 2)


def nan_logits(at):
    """Rows with a NaN among good logits, two of them, only four numbers, a +inf, and copies in front."""
    logits = torch.randn(6, 256, generator=torch.Generator().manual_seed(at))
    nan = float("nan")
    logits[0, at] = nan
    logits[1, [at, (at + 1) % 256]] = nan
    keep = logits[2, [3, 77, 130, 201]].clone()
    logits[2] = nan
    logits[2, [3, 77, 130, 201]] = keep
    logits[3, [at, 90]] = torch.tensor([nan, float("inf")])
    logits[4, :16] = 0.5
    logits[4, 200 + at % 50] = nan
    return logits


@pytest.mark.parametrize("at", [0, 31, 200, 255])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("form", ["bias", "groups", "both", "none"])
def test_nan_ranks_last_however_experts_are_chosen(form, scoring, at):
    """Choices by the scores of the other experts; the oracle leaves a NaN out of their sum."""
    logits = nan_logits(at)
    bias = 0.01 * torch.randn(256, generator=torch.Generator().manual_seed(1)) if form in ("bias", "both") else None
    groups = dict(num_groups=8, top_groups=3) if form in ("groups", "both") else {}
    for k in (1, 8):
        weights, ids = tnx.route_experts(logits.to(DEV), k, scoring=scoring,
                                         bias=None if bias is None else bias.to(DEV), **groups)
        w, want, _ = O.route_oracle(logits, k, scoring, bias, groups.get("num_groups", 1), groups.get("top_groups", 1))
        assert torch.equal(ids.cpu().long(), want)
        picked = logits.gather(1, want)
        good = [0, 1, 4, 5]
        assert torch.isfinite(picked[good]).all()
        torch.testing.assert_close(weights.cpu().double()[good], w[good], rtol=WEIGHT_RTOL, atol=1e-37)


def test_scores_next_to_a_nan_are_nan_unless_renormalised():
    logits = nan_logits(7)
    for kw in ({}, {"bias": torch.zeros(256, device=DEV)}):
        for scoring, lost in (("softmax", True), ("sigmoid", False)):
            w, ids = tnx.route_experts(logits.to(DEV), 4, scoring=scoring, renormalize=False, **kw)
            assert torch.isnan(w[0]).all().item() is lost
            assert 7 not in ids[0].tolist()
            assert torch.isfinite(tnx.route_experts(logits.to(DEV), 4, scoring=scoring, **kw)[0][0]).all()


def far_logits(dtype):
    """Logits at which a sigmoid or its complement leaves fp32."""
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(12, 24, generator=g)
    logits[0] -= 100.0
    logits[1] += 30.0
    logits[2] = logits[2] * 10 - 95
    logits[3] = logits[3] * 20 - 300
    logits[4, ::2] -= 120.0
    logits[5, ::3] += 60.0
    logits[6] = logits[6] * 0.5 - 700
    logits[7] = logits[7] * 40 - 720      # on both sides of where 64-bit scores end
    logits[8] -= 2000.0
    logits[9] = torch.finfo(dtype).min
    logits[10, 5:] = torch.finfo(dtype).min
    logits[11, 2:] = float("-inf")
    logits[11, :2] -= 150.0
    return logits.to(dtype)


@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [True, False])
def test_sigmoid_scores_far_from_zero(renormalize, biased, dtype):
    """Renormalised weights are ratios: they do not depend on whether fp32 holds the scores.  A score
    that is 0 in 64 bits is 0, a mask of the type's lowest value among them."""
    logits = far_logits(dtype)
    check(logits, 6, scoring="sigmoid", renormalize=renormalize, scale=1.5,
          **({"bias": torch.linspace(0.3, 0.0, 24)} if biased else {}))


@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("renormalize", [True, False])
def test_sigmoid_gradient_far_from_zero(renormalize, dtype):
    logits = far_logits(dtype)[[0, 1, 2, 3, 4, 5, 6]]
    dw = torch.randn(7, 6, generator=torch.Generator().manual_seed(2))
    leaf = logits.to(DEV).requires_grad_(True)
    weights, ids = tnx.route_experts(leaf, 6, scoring="sigmoid", renormalize=renormalize, scale=1.5)
    (grad,) = torch.autograd.grad(weights, leaf, dw.to(DEV))
    i = ids.cpu().long()
    ref = O.route_gradient_oracle(logits, i, dw, "sigmoid", renormalize, 1.5)
    # dl = 1.5 r (dw - sum dw r)(1 - s): every factor to 64 roundings of fp32 at most, the difference
    # against its terms' absolute values; one rounding to the type, subnormals of fp32 included
    z = logits.double()
    r = torch.sigmoid(z)
    if renormalize:
        r = r / r.gather(1, i).sum(1, keepdim=True)
    picks = torch.zeros_like(z).scatter_(1, i, 1.0)
    size = 1.5 * picks * r * torch.sigmoid(-z) * 2 * dw.abs().double().sum(1, keepdim=True)
    tol = 64 * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -133
    assert torch.isfinite(grad).all()
    assert ((grad.cpu().double() - ref).abs() <= tol).all()
    if renormalize:
        assert (grad[0].cpu()[i[0]] != 0).any()


def test_numbers_held_in_tensors_are_read_by_every_call():
    logits = torch.randn(4, 16, generator=torch.Generator().manual_seed(0)).to(DEV)
    scale, top_k = torch.tensor(1.0), torch.tensor(2)
    for value in (1, 3):
        scale.fill_(0.5 * value)
        top_k.fill_(value)
        want = tnx.route_experts(logits, value, scale=0.5 * value)
        got = tnx.route_experts(logits, top_k, scale=scale)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(ValueError, match="scale"):
        tnx.route_experts(logits, 2, scale=scale.requires_grad_(True))
