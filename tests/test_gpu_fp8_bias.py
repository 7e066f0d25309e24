"""Fp8Linear's bias in every type, in every kernel: added to the fp32 sums as it is, the result rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _sums(x, w, sw):
    return x.double() @ (w.double() * sw.double().repeat_interleave(128, 1)[:, : w.shape[1]].repeat_interleave(128, 0)[: w.shape[0]]).t()


def _case(M, N, K, seed=0):
    """x and a layer's weight whose sums are whole numbers below 2^20, exact in fp32 in any order, and a bias in eighths (eleven bits, which bf16 does not hold)."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(seed + N + K)
    x = torch.randint(-7, 8, (M, K), generator=gen, device="cuda").float()
    x[:, ::128] = 448.0  # (so that every scale is one)
    w = torch.randint(-3, 4, (N, K), generator=gen, device="cuda").float()
    w[:, ::128] = 0.0
    sw = torch.randint(-1, 2, (-(-N // 128), -(-K // 128)), generator=gen, device="cuda").float().exp2()
    bias = torch.randint(-2047, 2048, (N,), generator=gen, device="cuda").float() / 8 + 0.0
    q, s = g.quantize_per_token_block(x, dtype=F8)
    assert torch.equal(s, torch.ones_like(s)) and torch.equal(q.float(), x)
    want = _sums(x, w, sw) + bias.double()
    assert float(want.abs().max()) < 2 ** 20
    return x, w.to(F8), sw, bias, want.float().bfloat16()


SHAPES = [(1, 1024, 4096), (1, 1, 16), (16, 8192, 8192), (13, 200, 272), (16, 4096, 14336), (9, 5003, 1040), (40, 2048, 8192), (64, 4096, 14336), (100, 1001, 6992), (130, 1030, 8208),
          (256, 512, 14336), (17, 264, 128), (200, 3001, 512), (600, 4096, 512), (2500, 5000, 512), (300, 10240, 1024)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_fp32_bias(M, N, K):
    import gemm_int8_b200 as g

    x, w, sw, bias, want = _case(M, N, K)
    assert N < 8 or not torch.equal(bias.bfloat16().float(), bias)
    assert torch.equal(g.Fp8Linear(w, sw, bias)(x), want)
    wide = torch.full((N + 9,), float("nan"), device="cuda")
    for at in (1, 2, 4):  # (views at other alignments, NaN around them)
        wide[at : at + N] = bias
        assert torch.equal(g.Fp8Linear(w, sw, wide[at : at + N])(x), want)
        wide[at : at + N] = float("nan")
    assert torch.equal(g.Fp8Linear(w, sw, bias[:, None].expand(N, 2)[:, 0])(x), want)
    g.check_device()


@pytest.mark.parametrize("variant", ["pair", "dense_bn256", "dense_bn128", "dense_bn64"])
@pytest.mark.parametrize("M,N,K", [(17, 136, 272), (200, 301, 1040), (520, 776, 640)])
def test_fp32_bias_in_every_tile(M, N, K, variant):
    import gemm_int8_b200 as g

    x, w, sw, bias, want = _case(M, N, K)
    layer = g.Fp8Linear(w, sw, bias)
    g.force_variant(variant)
    try:
        out = layer(x)
    finally:
        g.force_variant(None)
    assert torch.equal(out, want)


@pytest.mark.parametrize("M,N,K", [(4, 264, 512), (40, 264, 512), (300, 520, 640)])
def test_other_types_of_bias(M, N, K):
    """bf16 as it is; fp16 and fp64 by way of fp32; a Parameter fused or, where it is differentiated, added to the product's rounded result."""
    import gemm_int8_b200 as g

    x, w, sw, bias, want = _case(M, N, K)
    assert torch.equal(bias.half().float(), bias)
    assert torch.equal(g.Fp8Linear(w, sw, bias.half())(x), want) and torch.equal(g.Fp8Linear(w, sw, bias.double())(x), want)
    rounded = bias.bfloat16()
    assert torch.equal(g.Fp8Linear(w, sw, rounded)(x), (_sums(x, w, sw) + rounded.double()).float().bfloat16())
    plain = g.Fp8Linear(w, sw)(x)
    parameter = g.Fp8Linear(w, sw, torch.nn.Parameter(bias.clone()))
    with torch.no_grad():
        assert torch.equal(parameter(x), want)
    open_ = parameter(x)
    assert open_.requires_grad and torch.equal(open_.detach(), (plain.float() + bias).bfloat16())
    open_.float().sum().backward()
    assert torch.equal(parameter.bias.grad, torch.full((N,), float(M), device="cuda"))
    full = g.Fp8Linear(w, sw, torch.nn.Parameter(bias.clone()), out_dtype=torch.float32)(x)
    assert torch.equal(full.detach(), plain.float() + bias)  # (nothing is rounded behind the sum)


def test_captured_with_a_bias_that_changes():
    import gemm_int8_b200 as g

    x, w, sw, bias, want = _case(24, 520, 1040)
    layer = g.Fp8Linear(w, sw, bias.clone())
    layer(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    graph.replay()
    assert torch.equal(out, want)
    layer.bias.add_(64.125)
    graph.replay()
    assert torch.equal(out, layer(x)) and not torch.equal(out, want)
