"""Groups whose values fp32 cannot tell apart: decided as the definition in 64 bits decides them."""
import pytest
import torch

from test_gpu_experts_route import _check

pytestmark = pytest.mark.gpu


# (groups of whole lanes, of a lane, and those that are looked up through shared memory)
@pytest.mark.parametrize("E,groups,top_groups", [(64, 8, 4), (256, 8, 3), (64, 32, 9), (60, 5, 2), (72, 4, 1)])
@pytest.mark.parametrize("B", [64.0, 256.0, 4096.0])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sums_that_cancel(E, groups, top_groups, B, scoring):
    """Every group's two largest choices are about B and -B: their sum is of the order of the scores, its fp32 error of the order of an ulp of B, and
    the exact sums lie within that of one another."""
    gen = torch.Generator().manual_seed(E + int(B))
    size = E // groups
    bias = torch.full((groups, size), -4.0 * B)
    bias[:, 0], bias[:, 1] = B, -B
    logits = torch.randn(groups, size, generator=gen)
    logits[:, 0], logits[:, 1] = 0.3, -0.2
    # scores that differ by half an ulp of B or so
    spread = 2.0 ** -24 * B * (4 if scoring == "sigmoid" else E)
    logits = logits.reshape(1, E) + spread * torch.randn(150, E, generator=gen)
    k = min(6, top_groups * size)
    _check(logits, k, scoring=scoring, bias=bias.reshape(E), groups=groups, top_groups=top_groups, group_score="top2")


@pytest.mark.parametrize("E,groups", [(64, 8), (32, 8), (60, 5), (72, 4)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masks_and_favours_of_the_largest_magnitude(E, groups, group_score, scoring):
    """A bias of fp32's lowest value masks all but one group: finite choices, whose groups are kept (the lower index first) and whose experts are chosen
    where nothing better is left, although the sum of two of them is beyond fp32.  The same for biases of the largest value."""
    gen = torch.Generator().manual_seed(E)
    size, top = E // groups, torch.finfo(torch.float32).max
    logits = torch.randn(20, E, generator=gen)
    bias = torch.full((groups, size), -top)
    bias[2] = torch.randn(size, generator=gen) * 0.1
    for top_groups in (1, 2, groups - 1):
        _check(logits, min(32, size * top_groups), scoring=scoring, bias=bias.reshape(E), groups=groups, top_groups=top_groups, group_score=group_score)
    bias = torch.randn(groups, size, generator=gen)
    bias[:, 0], bias[:, 1] = top, top * torch.linspace(0.1, 0.9, groups)
    _check(logits, min(2 * size, 8), scoring=scoring, bias=bias.reshape(E), groups=groups, top_groups=2, group_score=group_score)
