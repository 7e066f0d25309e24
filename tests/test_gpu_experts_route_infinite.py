"""Infinite logits: +inf counts as the largest finite value, so that a softmax shares its weight among the infinite ones."""
import math

import pytest
import torch

import experts_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,groups,top_groups,group_score", [(16, 1, 1, "max"), (64, 8, 2, "max"), (64, 8, 2, "top2"), (60, 5, 2, "top2")])
@pytest.mark.parametrize("renormalize", [False, True])
def test_infinite_logits(E, groups, top_groups, group_score, scoring, biased, renormalize, dtype):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(E)
    logits = torch.randn(6, E, generator=gen).to(dtype)
    logits[0, 5] = math.inf
    logits[1, 2], logits[1, 9] = math.inf, math.inf
    logits[2] = math.inf
    logits[3, ::3] = math.inf
    logits[3, 1::3] = -math.inf
    logits[4, 7], logits[4, 8] = math.inf, math.nan
    bias = torch.randn(E, generator=gen) * 0.1 if biased else None
    w, e = g.route_experts(logits.cuda(), 4, scoring=scoring, bias=None if bias is None else bias.cuda(), groups=groups, top_groups=top_groups,
                           group_score=group_score, renormalize=renormalize)
    # (the largest value of fp32: above all finite bf16 logits, and equal to none of the finite ones here)
    finite = torch.where(logits.float() == math.inf, torch.finfo(torch.float32).max, logits.float())
    w_ref, e_ref = R.route(finite, 4, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_score=group_score, renormalize=renormalize)
    assert torch.equal(e.cpu(), e_ref)
    # scores of finite logits within 10 of one another or 0 beside the infinite ones: expf 2 ulp and its argument, twice, and 40 roundings
    rel = 2 * (2 ** -22 + 10 * 2 ** -24) + 40 * 2 ** -24
    assert ((w.cpu().double() - w_ref).abs() <= rel * w_ref).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups,group_score", [(8, 1, 1, "max"), (64, 1, 1, "max"), (64, 8, 2, "max"), (64, 8, 2, "top2"), (60, 5, 2, "top2"), (72, 4, 1, "max")])
def test_infinite_biases(E, groups, top_groups, group_score, scoring):
    """A bias of +inf always chooses its expert, the lower index first; the weights do not see it."""
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(E)
    logits = torch.randn(9, E, generator=gen)
    logits[0, 3] = -math.inf
    for favoured in ([3], [3, 5], [1, 2, 3, E - 1], list(range(0, E, 2)), list(range(E))):
        bias = torch.randn(E, generator=gen) * 0.1
        bias[favoured] = math.inf
        w, e = g.route_experts(logits.cuda(), 4, scoring=scoring, bias=bias.cuda(), groups=groups, top_groups=top_groups, group_score=group_score)
        w_ref, e_ref = R.route(logits, 4, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_score=group_score)
        assert torch.equal(e.cpu(), e_ref)
        rel = 2 * (2 ** -22 + 10 * 2 ** -24) + 40 * 2 ** -24  # (as above)
        assert ((w.cpu().double() - w_ref).abs() <= rel * w_ref).all()
