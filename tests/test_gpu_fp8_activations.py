"""What Fp8Linear makes of the types it is given and asked for: fp16 activations by way of bf16, or in full as fp32; results rounded to bf16 and then cast."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(4, 264, 512), (40, 264, 1040), (300, 520, 640)])
def test_types_in_and_out(M, N, K):
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(K)
    w = torch.randn(N, K, generator=gen, device="cuda") * 0.05
    bias = torch.randn(N, generator=gen, device="cuda")
    layer, wide = g.Fp8Linear.from_float(w, bias), g.Fp8Linear.from_float(w, bias, out_dtype=torch.float32)
    x = R.outliers(gen, M, K, torch.float16)
    assert torch.equal(layer(x), layer(x.bfloat16()))
    q, s = g.quantize_per_token_block(x.float(), dtype=R.F8)
    want, err = R.product(q, layer.weight_q, s, layer.weight_scale)
    want = want + bias.double()
    out = layer(x.float())
    assert out.dtype == torch.bfloat16 and not torch.equal(out, layer(x))
    R.check_bf16(out, want, err + want.abs() * 2.0 ** -24)
    assert wide(x.float()).dtype == torch.float32 and torch.equal(wide(x.float()), out.float())
