"""swiglu_quantize against 64 bits, and the e4m3 form of quantize_per_token_block bit for bit against torch."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu
F8 = R.F8
FORMS = [("block", torch.int8), ("token", torch.int8), ("block", F8)]


def _check(gate_up, scales, dtype):
    import gemm_int8_b200 as g

    q, s = g.swiglu_quantize(gate_up, scales=scales, dtype=dtype)
    v, err = R.swiglu(gate_up)
    R.check_quantised(q, s, v, err, dtype, scales == "block")
    return q, s


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N", [(1, 16), (1, 128), (3, 144), (7, 1024), (16, 14336), (5, 6992), (1, 8192), (2, 8208), (1, 16400), (2, 28672), (2, 57344), (1, 131056),
                                 (777, 1408), (2000, 256), (300, 11008)])
def test_sizes_and_types(M, N, x, scales, dtype):
    gen = torch.Generator(device="cuda").manual_seed(M + N)
    _check((1.5 * R.outliers(gen, M, 2 * N, torch.float32)).to(x), scales, dtype)


@pytest.mark.parametrize("scales,dtype", FORMS)
def test_magnitudes(scales, dtype):
    """Gates from far below -88 (where exp overflows fp32) to far above, ups of zero and of large values, rows of zeros."""
    N = 640
    g = torch.linspace(-200, 200, N, device="cuda").repeat(6, 1)
    u = torch.randn(6, N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    g[1], u[2], u[3], g[4] = -100.0, 0.0, u[3] * 1e30, g[4] * 1e-30
    q, s = _check(torch.cat([g, u], 1), scales, dtype)
    assert torch.equal(s[2], torch.ones_like(s[2])) and not q[2].float().any()


@pytest.mark.parametrize("scales,dtype", FORMS)
def test_nan_and_infinity_show_in_the_scales(scales, dtype):
    import gemm_int8_b200 as g

    N = 512
    gu = torch.randn(5, 2 * N, device="cuda")
    gu[1, 200], gu[2, N + 200], gu[3, 200] = float("nan"), float("inf"), float("-inf")  # (-inf * 0 is NaN, as in torch)
    gu[2, 200] = 1.0
    q, s = g.swiglu_quantize(gu, scales=scales, dtype=dtype)
    s = s.reshape(5, -1)
    at = 200 // 128 if scales == "block" else 0
    assert torch.isnan(s[1, at]) and torch.isinf(s[2, at]) and torch.isnan(s[3, at])
    assert torch.isfinite(s[[0, 4]]).all() and (scales == "token" or torch.isfinite(s[:, [0, 2, 3]]).all())


def test_views_empty_and_refusals():
    import gemm_int8_b200 as g

    big = torch.randn(20, 2051, device="cuda").bfloat16()
    for x in (big[:, 3:1027], big[::3, 1024:2048], big[:, :20].t().contiguous().t()[:, :16].repeat(1, 2)):
        q, s = _check(x, "block", torch.int8)
        assert all(torch.equal(a, b) for a, b in zip((q, s), g.swiglu_quantize(x.contiguous())))
    q, s = g.swiglu_quantize(torch.empty(0, 512, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    q, s = g.swiglu_quantize(torch.empty(3, 0, device="cuda"), scales="token")
    assert q.shape == (3, 0) and s.shape == (3,)
    x = torch.randn(4, 512, device="cuda")
    for f in (lambda: g.swiglu_quantize(x.cpu()), lambda: g.swiglu_quantize(x.half()), lambda: g.swiglu_quantize(x[0]), lambda: g.swiglu_quantize(x[:, :511]),
              lambda: g.swiglu_quantize(x[:, :48]), lambda: g.swiglu_quantize(torch.empty(1, 2 * 131072, device="cuda"))):
        with pytest.raises(RuntimeError):
            f()
    for kw in ({"scales": "row"}, {"dtype": torch.float16}, {"scales": "token", "dtype": F8}):
        with pytest.raises(ValueError):
            g.swiglu_quantize(x, **kw)


@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 8), (1, 16), (1, 128), (3, 136), (5, 1000), (17, 4096), (2, 28672), (1000, 1408), (4099, 256)])
def test_e4m3_quantiser_bit_for_bit(M, K, x):
    import gemm_int8_b200 as g
    from gemm_int8_b200 import quant

    gen = torch.Generator(device="cuda").manual_seed(M * K)
    for scale in (1.0, 1e-18, 3e-22, 1e-36, 1e34):  # (scales below 1e-20 and above 1e30 take another path)
        a = (scale * R.outliers(gen, M, K, torch.float32)).to(x)
        q, s = g.quantize_per_token_block(a, dtype=F8)
        want_q, want_s = quant.quantize_per_token_block(a.float(), dtype=F8)
        assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


def test_e4m3_quantiser_between_two_numbers():
    """Quotients that lie between two e4m3 numbers exactly, or next to it by one unit of fp32 on either side."""
    import gemm_int8_b200 as g
    from gemm_int8_b200 import quant

    codes = torch.arange(0, 127, dtype=torch.uint8, device="cuda")
    v = codes[:126].view(F8).float()
    mid = (v + codes[1:].view(F8).float()) / 2
    mid = torch.cat([mid, torch.zeros(1, device="cuda"), torch.full((1,), 448.0, device="cuda")])
    rows = []
    gen = torch.Generator(device="cuda").manual_seed(5)
    for s in torch.rand(4000, generator=gen, device="cuda").mul(4).exp2().tolist() + [1.0, 0.75, 1.9999999]:
        t = mid * s
        rows += [t, torch.nextafter(t, t + 1), torch.nextafter(t, t - 1)]
    a = torch.stack(rows)
    q, s = g.quantize_per_token_block(a, dtype=F8)
    want_q, want_s = quant.quantize_per_token_block(a, dtype=F8)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


def test_e4m3_quantiser_nan_infinity_zeros():
    import gemm_int8_b200 as g
    from gemm_int8_b200 import quant

    a = torch.randn(8, 512, device="cuda")
    a[0, 130], a[1, 130], a[2, 128:256], a[3] = float("nan"), float("inf"), 0.0, -0.0
    for row, top in ((4, 1e-44), (5, 2e-43), (6, 1e-40), (7, 3e38)):  # scales of zero, subnormal scales, the largest
        a[row] = top
        a[row, ::3] = 0.0
    q, s = g.quantize_per_token_block(a, dtype=F8)
    want_q, want_s = quant.quantize_per_token_block(a, dtype=F8)
    assert torch.equal(torch.nan_to_num(s, -1.0, -2.0), torch.nan_to_num(want_s, -1.0, -2.0)) and torch.equal(torch.isnan(q.float()), torch.isnan(want_q.float()))
    assert torch.equal(torch.nan_to_num(q.float()), torch.nan_to_num(want_q.float()))
    assert torch.isfinite(q[2:].float()).all() and torch.equal(s[4], torch.ones_like(s[4])) and not q[4].float().any()
    for dtype in (torch.int8, F8):
        q, s = g.swiglu_quantize(torch.cat([torch.full((1, 128), 1e-22, device="cuda"), torch.full((1, 128), 1e-22, device="cuda")], 1), dtype=dtype)
        assert torch.equal(s, torch.ones_like(s)) and not q.float().any()
    with pytest.raises(ValueError):
        g.quantize_per_token_block(a, dtype=torch.float8_e5m2)
    with pytest.raises(RuntimeError):
        g.quantize_per_token_block(a[:, :12], dtype=F8)
