"""rms_norm_quantize against 64 bits: types, widths, batches, values that fp32 squares cannot hold, padding, NaN, views."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu
F8 = R.F8
FORMS = [("block", torch.int8), ("token", torch.int8), ("block", F8)]


def _check(x, weight, residual, eps, scales, dtype):
    import gemm_int8_b200 as g

    got = g.rms_norm_quantize(x, weight, residual, eps, scales=scales, dtype=dtype)
    v, h = R.norm(x, weight, residual, eps)
    R.check_quantised(got[0], got[1], v, v.abs() * R.NORM_REL, dtype, scales == "block")
    if residual is None:
        assert len(got) == 2
    else:
        total = x.float() + residual.float()
        assert got[2].dtype == residual.dtype and torch.equal(got[2], total.to(residual.dtype))
    return got


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("x,weight", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
def test_types(x, weight, residual, scales, dtype):
    gen = torch.Generator(device="cuda").manual_seed(7)
    for M, H in [(5, 4096), (3, 1040)]:
        a = R.outliers(gen, M, H, x)
        r = None if residual is None else (2 * torch.randn(M, H, generator=gen, device="cuda")).to(residual)
        w = (1 + 0.2 * torch.randn(H, generator=gen, device="cuda")).to(weight)
        _check(a, w, r, 1e-5, scales, dtype)


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("M,H", [(1, 16), (1, 128), (7, 112), (9, 144), (1, 256), (17, 272), (33, 512), (8, 1024), (1, 1040), (2, 2048), (5, 5120), (3, 6992), (1, 8192),
                                 (2, 8208), (300, 8192), (1, 14336), (2, 16384), (1, 16400), (2, 28672), (3, 32768), (1000, 640), (4099, 128)])
def test_sizes(M, H, scales, dtype):
    gen = torch.Generator(device="cuda").manual_seed(M * 131 + H)
    _check(R.outliers(gen, M, H, torch.bfloat16), torch.randn(H, generator=gen, device="cuda").bfloat16(), R.outliers(gen, M, H, torch.bfloat16), 1e-6, scales, dtype)


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("M,H", [(2, 16400), (2, 28672), (1, 32768), (400, 16384)])
def test_wide_fp32(M, H, scales, dtype):
    gen = torch.Generator(device="cuda").manual_seed(H)
    _check(R.outliers(gen, M, H, torch.float32), torch.randn(H, generator=gen, device="cuda"), R.outliers(gen, M, H, torch.float32), 1e-6, scales, dtype)


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("H", [256, 4096])
def test_padding_and_magnitudes(H, scales, dtype):
    """Rows of zeros, of fp32's largest values, of small ones next to eps, side by side."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(12, H, generator=gen, device="cuda")
    for row, m in enumerate([0.0, 1.0, 1e-3, 1e-20, 1e-38, 1e15, 1e17, 1e18, 1e25, 1e30, 3e37, 1e-6]):
        x[row] *= m
    w = torch.randn(H, generator=gen, device="cuda")
    w[: H // 2] = 0
    q, s = _check(x, w, None, 1e-12, scales, dtype)
    assert torch.equal(s[0], torch.ones_like(s[0])) and not q[0].float().any()
    zero = torch.zeros(12, H, device="cuda", dtype=torch.bfloat16)
    _check(x, w, zero, 1e-12, scales, dtype)


@pytest.mark.parametrize("scales,dtype", FORMS)
def test_nan_and_infinity_show_in_the_scales(scales, dtype):
    import gemm_int8_b200 as g

    H = 1024
    x = torch.randn(6, H, device="cuda")
    x[1, 300], x[2, 300], x[3, 5], w = float("nan"), float("inf"), float("-inf"), torch.ones(H, device="cuda")
    q, s = g.rms_norm_quantize(x, w, scales=scales, dtype=dtype)
    s = s.reshape(6, -1)
    assert torch.isnan(s[1]).all()
    for row, at in ((2, 300), (3, 5)):  # inf / inf in its own block; every other value is 0
        hit = s[row, at // 128 if scales == "block" else 0]
        assert torch.isnan(hit)
    clean = g.rms_norm_quantize(x[[0, 4, 5]], w, scales=scales, dtype=dtype)
    assert torch.equal(clean[0].view(torch.uint8), q[[0, 4, 5]].view(torch.uint8)) and torch.equal(clean[1].reshape(3, -1), s[[0, 4, 5]])


def test_views_and_batches():
    """Column slices, offsets that break 16-byte alignment, transposed memory, an expanded residual; a row's result does not depend on its batch."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(11)
    big = torch.randn(40, 3 * 512 + 3, generator=gen, device="cuda").bfloat16()
    w = torch.randn(600, generator=gen, device="cuda").bfloat16()[5:517]
    for x in (big[:, 512:1024], big[:, 1:513], big[::2, 3:515], big[:, :40].t().contiguous().t()[:, :32].repeat(1, 16)):
        r = big[:1, 7:519].expand(x.shape)
        got = _check(x, w, r, 1e-5, "block", torch.int8)
        again = g.rms_norm_quantize(x.contiguous(), w.contiguous(), r.contiguous(), 1e-5)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    x = R.outliers(gen, 700, 2048, torch.bfloat16)
    w = torch.randn(2048, generator=gen, device="cuda")
    many = g.rms_norm_quantize(x, w, x, dtype=F8)
    one = g.rms_norm_quantize(x[417:418], w, x[417:418], dtype=F8)
    assert all(torch.equal(a[417:418].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(many, one))


def test_empty():
    import gemm_int8_b200 as g

    w = torch.ones(256, device="cuda")
    for residual in (None, torch.empty(0, 256, device="cuda")):
        got = g.rms_norm_quantize(torch.empty(0, 256, device="cuda"), w, residual)
        assert got[0].shape == (0, 256) and got[1].shape == (0, 2) and (residual is None or got[2].shape == (0, 256))
    q, s = g.rms_norm_quantize(torch.empty(4, 0, device="cuda"), torch.empty(0, device="cuda"))
    assert q.shape == (4, 0) and s.shape == (4, 0)
    q, s = g.rms_norm_quantize(torch.empty(4, 0, device="cuda"), torch.empty(0, device="cuda"), scales="token")
    assert q.shape == (4, 0) and torch.equal(s, torch.ones(4, device="cuda"))


def test_refusals():
    import gemm_int8_b200 as g

    x, w = torch.randn(4, 256, device="cuda"), torch.ones(256, device="cuda")
    bad = [lambda: g.rms_norm_quantize(x.cpu(), w), lambda: g.rms_norm_quantize(x.half(), w), lambda: g.rms_norm_quantize(x[0], w), lambda: g.rms_norm_quantize(x, w[:128]),
           lambda: g.rms_norm_quantize(x, w.half()), lambda: g.rms_norm_quantize(x, w.cpu()), lambda: g.rms_norm_quantize(x, w, x[:2]), lambda: g.rms_norm_quantize(x, w, x.half()),
           lambda: g.rms_norm_quantize(x[:, :24], w[:24]), lambda: g.rms_norm_quantize(x, w, eps=0.0), lambda: g.rms_norm_quantize(x, w, eps=float("nan")),
           lambda: g.rms_norm_quantize(torch.empty(1, 32784, device="cuda"), torch.empty(32784, device="cuda"))]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    for kw in ({"scales": "row"}, {"dtype": torch.float16}, {"scales": "token", "dtype": F8}):
        with pytest.raises(ValueError):
            g.rms_norm_quantize(x, w, **kw)
