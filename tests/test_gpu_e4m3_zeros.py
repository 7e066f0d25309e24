"""Zeros of either sign in the e4m3 quantiser: the codes are those of the torch rule, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [1.0, 1e-18, 1e-24, 1e33])  # (scales below 1e-20 and above 1e30 take another path)
def test_sign_of_zero(top, x):
    import gemm_int8_b200 as g
    from gemm_int8_b200 import quant

    gen = torch.Generator(device="cuda").manual_seed(3)
    a = torch.randn(40, 1040, generator=gen, device="cuda") * top
    a[:, ::3] = -0.0
    a[:, 1::3] = 0.0
    a[7], a[8] = -0.0, 0.0
    a[9, ::5] = -top * 1e-9  # (quotients that round to zero from below)
    a = a.to(x)
    q, s = g.quantize_per_token_block(a, dtype=F8)
    want_q, want_s = quant.quantize_per_token_block(a.float(), dtype=F8)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
