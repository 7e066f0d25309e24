"""A layer whose experts are held by several ranks, with groups, bias and more pairs than one CTA groups."""
import pytest
import torch

import experts_reference as R
from test_gpu_experts_layer import _step_by_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k", [(40, 4), (1200, 8)])
@pytest.mark.parametrize("ranks", [2, 4])
def test_ranks_with_groups_and_bias(T, k, ranks):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(T + ranks)
    E, H, inner = 64, 144, 80
    held = E // ranks
    router = dict(scoring="sigmoid", bias=(torch.randn(E, generator=gen) * 0.1).cuda(), groups=8, top_groups=4, group_score="top2", scale=2.5)
    whole = g.Int8Experts.from_float(torch.randn(E, 2 * inner, H, generator=gen).cuda() * H ** -0.5, torch.randn(E, H, inner, generator=gen).cuda() * inner ** -0.5, k, **router)
    x, logits = torch.randn(T, H, generator=gen).bfloat16().cuda(), torch.randn(T, E, generator=gen).cuda()
    add = torch.randn(T, H, generator=gen).bfloat16().cuda()
    total, size = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for a in range(0, E, held):
        cut = slice(a, a + held)
        part = g.Int8Experts(whole.gate_up_q[cut], whole.gate_up_scale[cut], whole.down_q[cut], whole.down_scale[cut], k, first_expert=a, **router)
        share = part(x, logits, add if a == 0 else None)
        assert torch.equal(share, _step_by_step(part, x, logits, add if a == 0 else None))
        total, size = total + share.double(), size + share.double().abs()
    want = whole(x, logits, add)
    assert torch.equal(want, _step_by_step(whole, x, logits, add))
    # the magnitudes that the sums add up (a row of y does not depend on the rank that computes it)
    weights, experts = g.route_experts(logits, k, "sigmoid", router["bias"], 8, 4, "top2", True, 2.5)
    offsets, slots, places = g.group_by_expert(experts, E)
    x_q, x_scale = g.quantize_per_token(x)
    h_q, h_scale = g.quantize_per_token(g.matmul_experts_swiglu(x_q, whole.gate_up_q, x_scale, whole.gate_up_scale, offsets, slots, k))
    y = g.matmul_experts(h_q, whole.down_q, h_scale, whole.down_scale, offsets)
    _, magnitude = R.combine(y.cpu(), weights.cpu(), places.cpu(), add.cpu())
    # a share and the whole are rounded to bf16 once each (relative to the unrounded value), behind k + 1 fp32 roundings of at most that magnitude
    bound = 2 ** -8 * (1 + 2 ** -7) * (want.double().abs() + size) + 2 * (k + 1) * 2 ** -24 * magnitude.cuda()
    assert ((total - want.double()).abs() <= bound).all()
