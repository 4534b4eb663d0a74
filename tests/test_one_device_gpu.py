"""Tensors of a call that are on another device than q are refused before anything is launched."""
import pytest
import torch

import flash_attn_with_score_b200 as F

pytestmark = pytest.mark.gpu

OPERATORS = {
    "attention": lambda q, k, v: F.attention(q, k, v, True),
    "window": lambda q, k, v: F.attention_with_window(q, k, v, 10, 1),
    "scores": lambda q, k, v: F.attention_with_scores(q, k, v, True),
    "row sums": lambda q, k, v: F.attention_with_row_sum(q, k, v),
    "column sums": lambda q, k, v: F.attention_with_col_sum(q, k, v, True),
    "softmax sums": lambda q, k, v: F.attention_with_softmax_col_sum(q, k, v),
    "cross sums": lambda q, k, v: F.attention_cross_token_qk_sum(q, k, v, 5),
    "scores only": lambda q, k, v: F.compute_attention_scores(q, k),
}


@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("away", ["k", "v", "k and v"])
@pytest.mark.parametrize("grad", [False, True])
def test_keys_and_values(name, away, grad):
    if name == "scores only" and "k" not in away:
        pytest.skip("takes no values")
    q, k, v = (torch.randn((1, 2, 20, 64), device="cuda").half() for _ in range(3))
    if grad:
        q.requires_grad_()
    k, v = (x.cpu() if which in away else x for which, x in (("k", k), ("v", v)))
    with pytest.raises(AssertionError, match="one device"):
        OPERATORS[name](q, k, v)


def test_given_outputs_and_normalisers():
    q, k, v = (torch.randn((1, 2, 20, 64), device="cuda").half() for _ in range(3))
    host = torch.empty_like(q, device="cpu")
    with pytest.raises(AssertionError, match="one device"):
        F.attention_with_scores(q, k, v, out=host)
    with pytest.raises(AssertionError, match="one device"):
        F.attention_with_scores(q, k, v, scores=torch.empty((1, 2, 20, 20)))
    with pytest.raises(AssertionError, match="one device"):
        F.total_attention(q, k, torch.zeros((1, 2, 20)))
