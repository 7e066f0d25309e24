"""The router against its definition in 64 bits: experts equal, weights to fp32 rounding."""
import math

import pytest
import torch

import experts_reference as R

pytestmark = pytest.mark.gpu


def _check(logits, top_k, **kw):
    import gemm_int8_b200 as g

    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    w, e = g.route_experts(logits.cuda(), top_k, **dev)
    assert w.dtype == torch.float32 and e.dtype == torch.int32
    w_ref, e_ref = R.route(logits, top_k, **kw)
    assert torch.equal(e.cpu(), e_ref)
    # expf 2 ulp and its argument's rounding (the spread of a row's finite logits times 2^-24), once for the value and once for the sum; at most
    # 37 roundings in a sum over lanes; quotient, scale
    finite = torch.where(logits.float().isfinite(), logits.float(), torch.zeros(()))
    spread = float((finite.amax() - finite.amin()).clamp_min(finite.abs().amax())) if logits.numel() else 0.0
    rel = 2 * (2 ** -22 + spread * 2 ** -24) + 40 * 2 ** -24
    assert ((w.cpu().double() - w_ref).abs() <= rel * w_ref.abs() + 1e-37).all()


@pytest.mark.parametrize("T", [1, 3, 4, 130])
@pytest.mark.parametrize("E,k", [(1, 1), (8, 2), (31, 4), (33, 32), (60, 4), (64, 6), (128, 8), (160, 6), (256, 8), (320, 7), (512, 8), (1023, 5), (1024, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_plain(T, E, k, scoring):
    gen = torch.Generator().manual_seed(E * 7 + T)
    for dtype in (torch.float32, torch.bfloat16):
        logits = (torch.randn(T, E, generator=gen) * 2).to(dtype)
        for renorm in (True, False):
            _check(logits, k, scoring=scoring, renormalize=renorm, scale=2.5)
        _check(logits, k, scoring=scoring, bias=torch.randn(E, generator=gen) * 0.1)


@pytest.mark.parametrize("E,groups,top_groups,k", [(256, 8, 4, 8), (256, 8, 1, 8), (160, 8, 3, 6), (60, 5, 2, 4), (64, 32, 5, 6), (96, 3, 2, 9), (128, 16, 16, 8),
                                                   (1024, 32, 2, 32), (8, 2, 1, 4), (72, 4, 2, 8), (250, 5, 3, 8)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(E, groups, top_groups, k, group_score, scoring, biased):
    gen = torch.Generator().manual_seed(E + groups)
    bias = torch.randn(E, generator=gen) * 0.1 if biased else None
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.randn(37, E, generator=gen).to(dtype)
        _check(logits, k, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_score=group_score, scale=1.5)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_take_the_lowest_index(groups, top_groups, scoring, biased):
    logits = torch.randint(-2, 3, (64, 64), generator=torch.Generator().manual_seed(3)).float()
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    bias = torch.zeros(64) if biased else None
    for score in ("max", "top2"):
        _check(logits, 8, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_score=score)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_that_only_fp32_sees(scoring):
    """Pairs of experts whose biased scores differ by less than fp32 resolves, in either direction."""
    E = 64
    gen = torch.Generator().manual_seed(11)
    logits = torch.randn(50, E, generator=gen)
    score = torch.softmax(logits.double(), 1) if scoring == "softmax" else torch.sigmoid(logits.double())
    for t in range(50):
        # a bias that makes the best two of this token's scores equal up to its own rounding to fp32
        order = score[t].argsort(descending=True)
        bias = torch.zeros(E)
        bias[order[1]] = (score[t, order[0]] - score[t, order[1]]).float()
        _check(logits[t:t + 1], 2, scoring=scoring, bias=bias, renormalize=False)
        _check(logits[t:t + 1], 1, scoring=scoring, bias=bias, groups=8, top_groups=1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2), (8, 3)])
def test_masked_experts(scoring, biased, groups, top_groups):
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(8, 48, generator=gen)
    bias = torch.randn(48, generator=gen) * 0.1 if biased else None
    logits[0] = -math.inf                       # nothing left
    logits[1, 1:] = -math.inf                   # one left
    logits[2] = math.nan
    logits[3, ::3] = math.nan
    logits[4, 5:] = -math.inf
    logits[5, :40] = -math.inf                  # whole groups
    logits[6, ::2] = torch.finfo(torch.float32).min
    if biased:
        bias[7] = -math.inf
        bias[20] = math.nan
    for score in ("max", "top2"):
        _check(logits, 5, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_score=score)


def test_scores_far_below_one():
    """Sigmoid scores that fp32 cannot hold still have weights."""
    logits = -100.0 - torch.rand(4, 32, generator=torch.Generator().manual_seed(1))
    _check(logits, 4, scoring="sigmoid")
    _check(logits + 90.0, 4, scoring="sigmoid")


def test_infinite_logits_stay_in_bounds():
    import gemm_int8_b200 as g

    logits = torch.randn(4, 64, device="cuda")
    logits[0, 5] = math.inf
    logits[1, :] = math.inf
    for bias in (None, torch.zeros(64, device="cuda")):
        for scoring in ("softmax", "sigmoid"):
            _, e = g.route_experts(logits, 4, scoring=scoring, bias=bias)
            assert int(e.min()) >= -1 and int(e.max()) < 64
            if bias is None or scoring == "sigmoid":
                assert int(e[0, 0]) == 5


def test_strided_logits_and_many_tokens():
    import gemm_int8_b200 as g

    wide = torch.randn(5001, 96, generator=torch.Generator().manual_seed(2))
    w, e = g.route_experts(wide.cuda()[:, 7:71], 6)
    w2, e2 = g.route_experts(wide[:, 7:71].contiguous().cuda(), 6)
    assert torch.equal(w, w2) and torch.equal(e, e2)
    top = wide[:, 7:71].topk(6, dim=1)
    assert torch.equal(e.cpu().long(), top.indices)
    w, e = g.route_experts(torch.empty(0, 64, device="cuda"), 6)
    assert w.shape == (0, 6) and e.shape == (0, 6)
