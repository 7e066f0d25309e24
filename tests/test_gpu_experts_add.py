"""What is added to the weighted sum, in fp32 as in bf16."""
import pytest
import torch

import experts_reference as R
from test_gpu_experts_layer import _layer, _step_by_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,k", [(1, 8, 1), (1, 4096, 8), (3, 7, 2), (33, 2056, 5), (5, 1001, 32), (200, 520, 6)])
def test_sum_onto_fp32(T, N, k):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(T + N)
    y = torch.randn(T * k, N, generator=gen).bfloat16()
    weights = torch.randn(T, k, generator=gen) * 2.0 ** -6  # (what is added outweighs the sum: its bits are what counts)
    places = torch.randint(-1, T * k, (T, k), dtype=torch.int32, generator=gen)
    add = torch.randn(T, N, generator=gen)
    exact, size = R.combine(y, weights, places, add)
    flat = torch.empty(T * N + 1, device="cuda")  # (and off 16 bytes)
    flat[1:] = add.reshape(-1).cuda()
    for a in (add.cuda(), flat[1:].view(T, N), add.t().contiguous().cuda().t()):
        out = g.combine_experts(y.cuda(), weights.cuda(), places.cuda(), a).cpu().double()
        assert ((out - exact).abs() <= 2 ** -8 * exact.abs() + (k + 2) * 2 ** -24 * size).all()


def test_nothing_is_rounded_before_the_sum():
    """1 + 2^-9 is 1 in bf16, and 1 + 2^-9 + 2^-8 is nearer to 1 + 2^-7 than to 1."""
    import gemm_int8_b200 as g

    for N in (8, 7):
        out = g.combine_experts(torch.full((1, N), 2.0 ** -8, dtype=torch.bfloat16, device="cuda"), torch.ones(1, 1, device="cuda"),
                                torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1, N), 1 + 2.0 ** -9, device="cuda"))
        assert (out == 1 + 2.0 ** -7).all()


@pytest.mark.parametrize("T", [3, 200])
def test_layer_onto_other_types(T):
    import gemm_int8_b200 as g

    layer, gen = _layer(8, 64, 48, 2, seed=T)
    layer = layer.cuda()
    x, logits = torch.randn(T, 64, generator=gen).cuda(), torch.randn(T, 8, generator=gen).cuda()
    add = (torch.randn(T, 64, generator=gen) * 4).cuda()
    want = _step_by_step(layer, x, logits, add)
    assert torch.equal(layer(x, logits, add), want)
    assert torch.equal(layer(x, logits, add.double()), want)
    assert torch.equal(layer(x, logits, add.half()), _step_by_step(layer, x, logits, add.half().float()))
    assert torch.equal(layer(x, logits, add.bfloat16()), _step_by_step(layer, x, logits, add.bfloat16()))
    assert torch.equal(layer(x.double(), logits.double(), add), want)  # activations and logits of 64 bits go to fp32
