"""The 64-bit restatements of routing against values worked out by hand."""
import torch

from oracle import moe as O

nan, inf = float("nan"), float("inf")


def test_nan_ranks_last_and_the_others_keep_their_order():
    logits = torch.tensor([[nan, 1.0, 2.0, 3.0]])
    for kw in ({}, {"bias": torch.zeros(4)}, {"groups": 2, "top_groups": 1}):
        for scoring in ("softmax", "sigmoid"):
            w, ids, _ = O.route_oracle(logits, 2, scoring, **kw)
            assert ids.tolist() == [[3, 2]]
            if scoring == "softmax":
                torch.testing.assert_close(w, torch.softmax(torch.tensor([[3.0, 2.0]]).double(), 1))
    # scores of the other three are 0.09, 0.24, 0.67: a bias of 0.2 lifts the first past the second
    _, ids, _ = O.route_oracle(logits, 3, bias=torch.tensor([9.0, 0.2, 0.0, 0.0]))
    assert ids.tolist() == [[3, 1, 2]]
    w, _, _ = O.route_oracle(logits, 2, renormalize=False)
    assert torch.isnan(w).all()


def test_infinity_is_the_limit_of_a_large_logit():
    _, ids, _ = O.route_oracle(torch.tensor([[5.0, inf, 4.0, -inf]]), 4, bias=torch.zeros(4))
    assert ids.tolist() == [[1, 0, 2, 3]]
