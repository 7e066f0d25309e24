"""The experts' operators on views: bases off 16 bytes and strided arguments give what aligned, contiguous copies give, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _shifted(t):
    """The same values, contiguous, one element behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    out = flat[1:].view(t.shape)
    assert out.is_contiguous() and out.data_ptr() % 16 != 0
    return out


def _strided(t):
    """The same values, every other element of rows twice as long."""
    wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device)
    wide[..., ::2] = t
    return wide[..., ::2]


@pytest.mark.parametrize("E", [8, 64, 128, 160, 256, 512, 1024])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_router(E, dtype):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(E)
    logits, bias = torch.randn(133, E, generator=gen).to(dtype).cuda(), (torch.randn(E, generator=gen) * 0.1).cuda()
    for scoring in ("softmax", "sigmoid"):
        for kw in ({}, dict(groups=4, top_groups=2, group_score="top2", scale=2.5)):
            for b in (None, bias):
                want = g.route_experts(logits, 4, scoring, b, **kw)
                for l2, b2 in ((_shifted(logits), b), (_strided(logits), b), (logits, b if b is None else _shifted(b)), (_shifted(logits), b if b is None else _strided(b))):
                    assert all(torch.equal(x, y) for x, y in zip(g.route_experts(l2, 4, scoring, b2, **kw), want))


def test_grouping():
    import gemm_int8_b200 as g

    for T in (50, 3000):
        experts = torch.randint(-1, 12, (T, 5), dtype=torch.int32, generator=torch.Generator().manual_seed(T)).cuda()
        want = g.group_by_expert(experts, 9, 2)
        for e in (_shifted(experts), _strided(experts)):
            assert all(torch.equal(x, y) for x, y in zip(g.group_by_expert(e, 9, 2), want))


@pytest.mark.parametrize("T,k", [(9, 2), (300, 4)])
@pytest.mark.parametrize("N", [128, 130])
def test_products(T, k, N):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(T + N)
    E, K = 6, 272
    experts = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)]).int().cuda()
    offsets, slots, _ = g.group_by_expert(experts, E)
    x = torch.randint(-128, 128, (T, K), dtype=torch.int8, generator=gen).cuda()
    w = torch.randint(-128, 128, (E, N, K), dtype=torch.int8, generator=gen).cuda()
    sx, sw = torch.rand(T, generator=gen).cuda() * 0.01, torch.rand(E, N, generator=gen).cuda() * 0.01
    for f in (g.matmul_experts, g.matmul_experts_swiglu):
        want = f(x, w, sx, sw, offsets, slots, k)
        for change in (_shifted, _strided):
            assert torch.equal(f(x, w, sx, change(sw), offsets, slots, k), want)
            assert torch.equal(f(x, w, change(sx), sw, offsets, slots, k), want)
            assert torch.equal(f(x, w, sx, sw, change(offsets), change(slots), k), want)


@pytest.mark.parametrize("T,N,k", [(3, 8, 1), (40, 520, 6), (7, 2056, 3)])
def test_sum(T, N, k):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(N)
    y, add = torch.randn(T * k, N, generator=gen).bfloat16().cuda(), torch.randn(T, N, generator=gen).bfloat16().cuda()
    weights, places = torch.randn(T, k, generator=gen).cuda(), torch.randint(-1, T * k, (T, k), dtype=torch.int32, generator=gen).cuda()
    want, plain = g.combine_experts(y, weights, places, add), g.combine_experts(y, weights, places)
    for change in (_shifted, _strided):
        assert torch.equal(g.combine_experts(change(y), weights, places, add), want)
        assert torch.equal(g.combine_experts(y, change(weights), places, add), want)
        assert torch.equal(g.combine_experts(y, weights, change(places), add), want)
        assert torch.equal(g.combine_experts(y, weights, places, change(add)), want)
        assert torch.equal(g.combine_experts(change(y), change(weights), change(places)), plain)


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer(T, dtype):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(T)
    E, H, inner, k = 8, 144, 80, 3
    bias = (torch.randn(E, generator=gen) * 0.1).cuda()
    layer = g.Int8Experts.from_float(torch.randn(E, 2 * inner, H, generator=gen).cuda(), torch.randn(E, H, inner, generator=gen).cuda(), k, scoring="sigmoid", bias=bias)
    x, logits = torch.randn(T, H, generator=gen).to(dtype).cuda(), torch.randn(T, E, generator=gen).to(dtype).cuda()
    add = torch.randn(T, H, generator=gen).bfloat16().cuda()
    want = layer(x, logits, add)
    for change in (_shifted, _strided):
        assert torch.equal(layer(change(x), logits, add), want)
        assert torch.equal(layer(x, change(logits), add), want)
        assert torch.equal(layer(x, logits, change(add)), want)
        other = g.Int8Experts(layer.gate_up_q, change(layer.gate_up_scale), layer.down_q, change(layer.down_scale), k, scoring="sigmoid", bias=change(bias))
        assert torch.equal(other(x, logits, add), want)
