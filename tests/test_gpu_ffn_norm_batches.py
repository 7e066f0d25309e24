"""A row of rms_norm_quantize is what it is by itself, bit for bit, whatever the batch: small batches run in other forms of the kernel than large ones."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu
FORMS = [("block", torch.int8), ("token", torch.int8), ("block", R.F8)]


def _same(many, few, rows):
    for a, b in zip(many, few):
        assert torch.equal(a[rows].contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [16, 128, 256, 272, 512, 528, 1024, 1040, 2048, 4096, 6992, 8192])
def test_every_row_whatever_the_batch(H, residual, scales, dtype):
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(H)
    small = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    M = 2 * small + 77
    x = R.outliers(gen, M, H, torch.bfloat16 if H % 512 else torch.float32)
    r = None if residual is None else R.outliers(gen, M, H, residual)
    w = torch.randn(H, generator=gen, device="cuda")
    many = g.rms_norm_quantize(x, w, r, scales=scales, dtype=dtype)
    for a, b in ((0, small), (small, 2 * small), (2 * small, M), (417, 418), (M - 1, M)):
        _same(many, g.rms_norm_quantize(x[a:b], w, None if r is None else r[a:b], scales=scales, dtype=dtype), slice(a, b))


@pytest.mark.parametrize("H", [256, 1040, 8192])
def test_rows_whose_squares_overflow(H):
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(H)
    M = 700
    x = torch.randn(M, H, generator=gen, device="cuda") * 1e18
    w = torch.randn(H, generator=gen, device="cuda")
    many = g.rms_norm_quantize(x, w, dtype=R.F8)
    _same(many, g.rms_norm_quantize(x[300:400], w, dtype=R.F8), slice(300, 400))
    v, _ = R.norm(x, w, None, 1e-6)
    R.check_quantised(many[0], many[1], v, v.abs() * R.NORM_REL, R.F8, True)
