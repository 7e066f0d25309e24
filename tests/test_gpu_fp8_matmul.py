"""matmul_blockwise_fp8 and Fp8Linear against 64 bits, and bit for bit where fp32 sums are exact."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu
F8 = R.F8


def _operands(M, N, K, seed=0):
    from gemm_int8_b200 import quant

    gen = torch.Generator(device="cuda").manual_seed(seed + M + 3 * N + 7 * K)
    x_q, x_s = quant.quantize_per_token_block(R.outliers(gen, M, K, torch.float32), dtype=F8)
    w_q, w_s = quant.quantize_weight_block(torch.randn(N, K, generator=gen, device="cuda") * 0.02, dtype=F8)
    return x_q, w_q, x_s, w_s


SIZES = [(1, 1, 16), (1, 64, 128), (3, 130, 144), (16, 256, 256), (16, 4096, 4096), (13, 5003, 1040), (17, 64, 128), (17, 200, 272), (64, 4096, 1024), (100, 1001, 6992),
         (128, 256, 128), (129, 257, 384), (256, 8192, 512), (300, 4096, 4096), (512, 10240, 1024), (777, 5003, 6992), (1024, 4096, 4096), (2048, 8192, 1040), (33, 37, 28672)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(M, N, K):
    import gemm_int8_b200 as g

    ops = _operands(M, N, K)
    out = g.matmul_blockwise_fp8(*ops)
    assert out.dtype == torch.bfloat16 and out.shape == (M, N)
    R.check_bf16(out, *R.product(*ops))
    g.check_device()


@pytest.mark.parametrize("variant", ["pair", "dense_bn256", "dense_bn128", "dense_bn64"])
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (200, 300, 1040), (500, 776, 2048), (2100, 5000, 512)])
def test_every_tile(M, N, K, variant):
    import gemm_int8_b200 as g

    ops = _operands(M, N, K)
    g.force_variant(variant)
    try:
        out = g.matmul_blockwise_fp8(*ops)
    finally:
        g.force_variant(None)
    R.check_bf16(out, *R.product(*ops))
    g.check_device()


@pytest.mark.parametrize("M,N,K", [(4, 200, 512), (16, 320, 1040), (40, 200, 512), (130, 520, 384), (700, 2048, 640)])
@pytest.mark.parametrize("variant", [None, "pair", "dense_bn256", "dense_bn128", "dense_bn64"])
def test_exact_sums(M, N, K, variant):
    """Whole numbers whose sums stay below 2^24 and scales that are powers of two: every fp32 step is exact, so the result is the rounded sum."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randint(-15, 16, (M, K), generator=gen, device="cuda").float()
    w = torch.randint(-15, 16, (N, K), generator=gen, device="cuda").float()
    KB = -(-K // 128)
    sx = torch.randint(-1, 2, (M, KB), generator=gen, device="cuda").float().exp2()
    sw = torch.randint(-1, 2, (-(-N // 128), KB), generator=gen, device="cuda").float().exp2()
    x_q, w_q = x.to(F8), w.to(F8)
    assert torch.equal(x_q.float().clamp(-15, 15), x_q.float()) and torch.equal(x_q.float().round(), x_q.float())
    want, _ = R.product(x_q, w_q, sx, sw)
    assert float(want.abs().max()) < 2 ** 22
    g.force_variant(variant)
    try:
        out = g.matmul_blockwise_fp8(x_q, w_q, sx, sw)
    finally:
        g.force_variant(None)
    assert torch.equal(out, want.float().bfloat16())


@pytest.mark.parametrize("M,N,K", [(7, 136, 272), (200, 264, 512)])
def test_subnormal_codes(M, N, K):
    """Multiples of 2^-9, among them all of e4m3's subnormal numbers, which must not be flushed: exact sums of multiples of 2^-18."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randint(-15, 16, (M, K), generator=gen, device="cuda").float() * 2.0 ** -9
    w = torch.randint(-7, 8, (N, K), generator=gen, device="cuda").float() * 2.0 ** -9
    x_q, w_q = x.to(F8), w.to(F8)
    assert torch.equal(x_q.float(), x) and torch.equal(w_q.float(), w)
    one = torch.ones(max(M, -(-N // 128)), -(-K // 128), device="cuda")
    want = R.product(x_q, w_q, one[:M], one[: -(-N // 128)])[0]
    assert torch.equal(g.matmul_blockwise_fp8(x_q, w_q, one[:M], one[: -(-N // 128)]), want.float().bfloat16())


@pytest.mark.parametrize("M,N,K", [(1, 64, 28672), (16, 200, 2064), (9, 4096, 14336), (5, 1000, 4112), (16, 2048, 8192), (40, 2048, 8192), (64, 4096, 14336), (100, 1001, 6992),
                                   (33, 5003, 4096), (256, 512, 14336), (17, 100, 28672), (130, 1030, 8208), (1024, 1024, 8192), (64, 8192, 28672), (128, 8192, 8192)])
@pytest.mark.parametrize("bias", [False, True])
def test_split_k_blocks(M, N, K, bias):
    """Few tiles with long sums: the K blocks of a tile are shared out.  Exact sums, as above, so the result is the same whoever adds them up; the layer's bias is a whole number."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(K + N)
    KB = -(-K // 128)
    x_q = torch.randint(-7, 8, (M, K), generator=gen, device="cuda").float().to(F8)
    w_q = torch.randint(-7, 8, (N, K), generator=gen, device="cuda").float().to(F8)
    sx, sw = torch.randint(0, 2, (M, KB), generator=gen, device="cuda").float().exp2(), torch.randint(-1, 1, (-(-N // 128), KB), generator=gen, device="cuda").float().exp2()
    want = R.product(x_q, w_q, sx, sw)[0]
    assert float(want.abs().max()) < 2 ** 22
    if not bias:
        assert torch.equal(g.matmul_blockwise_fp8(x_q, w_q, sx, sw), want.float().bfloat16())
    else:  # the layer quantises what dequantises exactly: blocks whose largest magnitude is 448 times a power of two
        a = x_q.float()
        a[:, ::128] = 448.0
        b = torch.randint(-8, 9, (N,), generator=gen, device="cuda").float()
        q, s = g.quantize_per_token_block(a, dtype=F8)
        assert torch.equal(s, torch.ones_like(s)) and torch.equal(q.float(), a)
        want = R.product(q, w_q, s, sw)[0] + b.double()
        assert float(want.abs().max()) < 2 ** 23
        assert torch.equal(g.Fp8Linear(w_q, sw, b.bfloat16())(a), want.float().bfloat16())
    g.check_device()


@pytest.mark.parametrize("M,N", [(8, 64), (64, 256), (300, 512)])
def test_large_and_small_products_in_one_block(M, N):
    """Products of 448 x 448 that cancel and products of 1 beside them in the same K block: what is left is what fp32 sums keep."""
    import gemm_int8_b200 as g

    K = 256
    x, w = torch.ones(M, K, device="cuda"), torch.ones(N, K, device="cuda")
    x[:, :16], w[:, :16] = 448.0, 448.0
    x[:, 1:16:2] *= -1
    one = torch.ones(1, device="cuda")
    out = g.matmul_blockwise_fp8(x.to(F8), w.to(F8), one.expand(M, 2).contiguous(), one.expand(-(-N // 128), 2).contiguous())
    assert torch.equal(out, torch.full_like(out, 240.0))


@pytest.mark.parametrize("M", [5, 200])
def test_special_values(M):
    """NaN operands and scales reach the outputs that use them and no others; infinite and huge scales do what fp32 does."""
    import gemm_int8_b200 as g

    N, K = 264, 512
    x_q, w_q, x_s, w_s = _operands(M, N, K)
    base = g.matmul_blockwise_fp8(x_q, w_q, x_s, w_s)
    x2, s2 = x_q.clone(), x_s.clone()
    x2.view(torch.uint8)[2, 300] = 0x7F
    s2[3, 1] = float("nan")
    s2[4, 2] = float("inf")
    out = g.matmul_blockwise_fp8(x2, w_q, s2, w_s)
    assert torch.isnan(out[2]).all() and torch.isnan(out[3]).all() and not torch.isfinite(out[4]).any()
    rest = [m for m in range(M) if m not in (2, 3, 4)]
    assert torch.equal(out[rest], base[rest])
    w2 = w_q.clone()
    w2.view(torch.uint8)[130, 7] = 0xFF
    out = g.matmul_blockwise_fp8(x_q, w2, x_s, w_s)
    assert torch.isnan(out[:, 130]).all() and torch.equal(torch.cat([out[:, :130], out[:, 131:]], 1), torch.cat([base[:, :130], base[:, 131:]], 1))
    out = g.matmul_blockwise_fp8(x_q, w_q, x_s * 2.0 ** 100, w_s * 2.0 ** -100)
    assert torch.equal(out, base)


def test_scale_views_empty_and_refusals():
    import gemm_int8_b200 as g

    x_q, w_q, x_s, w_s = _operands(40, 300, 1040)
    base = g.matmul_blockwise_fp8(x_q, w_q, x_s, w_s)
    wide = torch.randn(40, 30, device="cuda")
    wide[:, 3:12] = x_s
    assert torch.equal(base, g.matmul_blockwise_fp8(x_q, w_q, wide[:, 3:12], w_s.t().contiguous().t()))
    assert g.matmul_blockwise_fp8(x_q[:0], w_q, x_s[:0], w_s).shape == (0, 300)
    assert g.matmul_blockwise_fp8(x_q, w_q[:0], x_s, w_s[:0]).shape == (40, 0)
    none = g.matmul_blockwise_fp8(x_q[:, :0].contiguous(), w_q[:, :0].contiguous(), x_s[:, :0], w_s[:, :0])
    assert none.shape == (40, 300) and not none.any()
    shifted = torch.empty(40 * 1040 + 1, dtype=torch.uint8, device="cuda")[1:].view(F8).view(40, 1040)
    bad = [lambda: g.matmul_blockwise_fp8(x_q.cpu(), w_q, x_s, w_s), lambda: g.matmul_blockwise_fp8(x_q.view(torch.int8), w_q.view(torch.int8), x_s, w_s),
           lambda: g.matmul_blockwise_fp8(x_q, w_q.float(), x_s, w_s), lambda: g.matmul_blockwise_fp8(x_q, w_q[:, :1024].contiguous(), x_s, w_s),
           lambda: g.matmul_blockwise_fp8(x_q, w_q, x_s[:, :8], w_s), lambda: g.matmul_blockwise_fp8(x_q, w_q, x_s, w_s.double()),
           lambda: g.matmul_blockwise_fp8(x_q[:, :1032].contiguous(), w_q[:, :1032].contiguous(), x_s, w_s), lambda: g.matmul_blockwise_fp8(x_q[::2], w_q, x_s[::2], w_s),
           lambda: g.matmul_blockwise_fp8(x_q.to(torch.float8_e5m2), w_q, x_s, w_s), lambda: g.matmul_blockwise_fp8(x_q[0], w_q, x_s, w_s),
           lambda: g.matmul_blockwise_fp8(shifted, w_q, x_s, w_s)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 512), (4, 136, 1040), (16, 8200, 256), (40, 1000, 384), (200, 3001, 512), (600, 10240, 1024), (2500, 5000, 512)])
def test_linear(M, N, K, x, bias):
    """The layer is its quantiser and its product; a bias is added before the rounding."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    w = torch.randn(N, K, generator=gen, device="cuda") * 0.02
    b = torch.randn(N, generator=gen, device="cuda").bfloat16() if bias else None
    layer = g.Fp8Linear.from_float(w, b)
    assert (layer.in_features, layer.out_features) == (K, N)
    a = R.outliers(gen, M, K, x)
    out = layer(a)
    q, s = g.quantize_per_token_block(a, dtype=F8)
    if not bias:
        assert torch.equal(out, g.matmul_blockwise_fp8(q, layer.weight_q, s, layer.weight_scale))
    want, err = R.product(q, layer.weight_q, s, layer.weight_scale)
    if bias:
        want = want + b.double()
        err = err + want.abs() * 2.0 ** -24
    R.check_bf16(out, want, err)
    g.check_device()


def test_linear_shapes_types_and_refusals():
    import gemm_int8_b200 as g

    w = torch.randn(264, 256, device="cuda") * 0.05
    layer = g.Fp8Linear.from_float(w, torch.randn(264, device="cuda"), out_dtype=torch.float32)
    x = torch.randn(2, 3, 256, device="cuda")
    out = layer(x)
    assert out.shape == (2, 3, 264) and out.dtype == torch.float32 and torch.equal(out.reshape(6, 264), layer(x.reshape(6, 256)))
    assert torch.equal(layer(x.half()), layer(x.half().bfloat16())) and torch.equal(layer(x.double()), layer(x))
    assert layer(x[:0]).shape == (0, 3, 264)
    assert torch.equal(layer(x.reshape(6, 256)[:, :].t().contiguous().t()), layer(x.reshape(6, 256)))
    parameter = g.Fp8Linear(layer.weight_q, layer.weight_scale, torch.nn.Parameter(torch.randn(264, device="cuda")))
    with torch.no_grad():
        fused = parameter(x)
    open_ = parameter(x)
    assert open_.requires_grad and torch.allclose(fused.float(), open_.float(), rtol=2 ** -6, atol=2 ** -6)
    with pytest.raises(ValueError):
        g.Fp8Linear(layer.weight_q.view(torch.int8), layer.weight_scale)
    for f in (lambda: layer(x.cpu()), lambda: layer(x[..., :128]), lambda: g.Fp8Linear(layer.weight_q, layer.weight_scale[:2])(x)):
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("M,N,K", [(20, 300, 272), (130, 520, 2064), (777, 640, 28672), (1024, 5003, 6992), (300, 9472, 6912), (40, 1024, 8320), (600, 4736, 4224)])
def test_scales_inside_a_wider_buffer(M, N, K):
    """Any number of K blocks, rows of scales at any stride: what lies behind the last row and the last column is NaN and reaches nothing."""
    import gemm_int8_b200 as g

    ops = _operands(M, N, K)
    want = g.matmul_blockwise_fp8(*ops)
    R.check_bf16(want, *R.product(*ops))
    for extra in (1, 3, 4):
        wide = []
        for s in ops[2:]:
            buf = torch.full((s.shape[0] + 3, s.shape[1] + extra), float("nan"), device="cuda")
            buf[: s.shape[0], : s.shape[1]] = s
            wide.append(buf[: s.shape[0], : s.shape[1]])
        assert torch.equal(g.matmul_blockwise_fp8(ops[0], ops[1], *wide), want)
    g.check_device()


@pytest.mark.parametrize("N,K", [(14336, 512), (4096, 4096), (9472, 640), (1000, 8320)])
def test_fewer_rows_than_a_tile(N, K):
    """Every number of rows up to a tile's gives the rows of the largest: bit for bit where the same tiles are taken, and right where K blocks are shared out otherwise."""
    import gemm_int8_b200 as g

    x_q, w_q, x_s, w_s = _operands(128, N, K)
    full = torch.full_like(x_q.view(torch.uint8), 0x7F).view(F8)  # NaN behind the rows that a call is given
    for M in (17, 18, 23, 24, 25, 31, 33, 40, 63, 65, 97, 121, 127, 128):
        full.view(torch.uint8)[:M] = x_q.view(torch.uint8)[:M]
        out = g.matmul_blockwise_fp8(full[:M], w_q, x_s[:M], w_s)
        R.check_bf16(out, *R.product(x_q[:M], w_q, x_s[:M], w_s))
    for variant in ("dense_bn128", "dense_bn64", "dense_bn256", "pair"):
        g.force_variant(variant)
        try:
            want = g.matmul_blockwise_fp8(x_q, w_q, x_s, w_s)
            for M in (1, 7, 17, 24, 100):
                assert torch.equal(g.matmul_blockwise_fp8(x_q[:M], w_q, x_s[:M], w_s), want[:M]), (variant, M)
        finally:
            g.force_variant(None)
    g.check_device()
