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


@pytest.mark.parametrize("E,groups,top_groups", [(60, 5, 2), (72, 4, 2), (250, 5, 3), (256, 8, 4)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_of_groups(E, groups, top_groups, group_score, scoring, biased):
    """Equal groups whatever way their values are looked up, and more equal candidates than a warp has lanes."""
    logits = torch.randint(-2, 3, (40, E), generator=torch.Generator().manual_seed(E)).float()
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    logits[2, :E // 2] = -float("inf")
    bias = torch.zeros(E) if biased else None
    for k in (1, 8, min(32, top_groups * E // groups)):
        _check(logits, k, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_score=group_score)


@pytest.mark.parametrize("E,groups", [(60, 5), (72, 4), (256, 8)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_groups_that_only_fp32_sees_as_equal(E, groups, group_score, scoring, biased):
    """The best two groups' values differ by less than fp32 resolves, in either direction: by a bias that makes them equal up to its own rounding, or
    (without one) by logits whose scores do."""
    gen = torch.Generator().manual_seed(E + 1)
    n = 1 if group_score == "max" else 2
    size = E // groups
    for t in range(20):
        logits = torch.randn(1, E, generator=gen)
        if biased:
            score = torch.softmax(logits.double(), 1) if scoring == "softmax" else torch.sigmoid(logits.double())
            by_group = score.reshape(groups, size).sort(dim=1, descending=True)
            value = by_group.values[:, :n].sum(1)
            best, next_best = value.topk(2).indices.tolist()
            bias = torch.zeros(groups, size)
            bias[next_best, by_group.indices[next_best, 0]] = (value[best] - value[next_best]).float()
            bias = bias.reshape(E)
        else:
            # the same logits in all groups, in other orders, one of them moved by an ulp or none
            bias = None
            row = torch.randn(size, generator=gen)
            logits = torch.stack([row[torch.randperm(size, generator=gen)] for _ in range(groups)]).reshape(1, E)
            i = int(torch.randint(0, E, (1,), generator=gen))
            logits[0, i] = torch.nextafter(logits[0, i], torch.tensor(float(t % 3 - 1) * 10))
        _check(logits, 4, scoring=scoring, bias=bias, groups=groups, top_groups=1, group_score=group_score)
