"""The weighted sum, and the layer that runs the operators one after the other."""
import pytest
import torch

import experts_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,k", [(1, 8, 1), (1, 4096, 8), (3, 7, 2), (33, 2056, 5), (5, 1001, 32), (200, 520, 6)])
@pytest.mark.parametrize("with_add", [False, True])
def test_combine(T, N, k, with_add):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(T + N)
    rows = T * k + 3
    y = torch.randn(rows, N, generator=gen).to(torch.bfloat16)
    weights = torch.randn(T, k, generator=gen)
    places = torch.randint(-1, rows, (T, k), dtype=torch.int32, generator=gen)
    places[0] = -1
    add = torch.randn(T, N, generator=gen).to(torch.bfloat16) if with_add else None
    out = g.combine_experts(y.cuda(), weights.cuda(), places.cuda(), None if add is None else add.cuda()).cpu().double()
    exact, size = R.combine(y, weights, places, add)
    assert ((out - exact).abs() <= 2 ** -8 * exact.abs() + (k + 2) * 2 ** -24 * size).all()
    if not with_add:
        assert (out[0] == 0).all()


def test_combine_leaves_out_what_has_no_row():
    """A place that is left out does not read y: infinities and NaN elsewhere stay elsewhere."""
    import gemm_int8_b200 as g

    y = torch.full((4, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    y[1] = 2.0
    places = torch.tensor([[1, -1], [-1, -1], [-7, 1], [4, 1]], dtype=torch.int32, device="cuda")
    weights = torch.tensor([[0.5, float("nan")]], device="cuda").repeat(4, 1)
    weights[2:, 1] = 0.5
    out = g.combine_experts(y, weights, places)
    assert torch.equal(out.cpu(), torch.tensor([1.0, 0.0, 1.0, 1.0], dtype=torch.bfloat16)[:, None].expand(4, 64))


def _layer(E, H, inner, k, seed, **router):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(seed)
    gate_up = torch.randn(E, 2 * inner, H, generator=gen) * H ** -0.5
    down = torch.randn(E, H, inner, generator=gen) * inner ** -0.5
    return g.Int8Experts.from_float(gate_up, down, k, **router), gen


def _step_by_step(layer, x, logits, add=None):
    import gemm_int8_b200 as g

    k, sigmoid, groups, top_groups, top2, renorm, scale = layer._router
    weights, experts = g.route_experts(logits, k, "sigmoid" if sigmoid else "softmax", layer.bias, groups, top_groups, "top2" if top2 else "max", renorm, scale)
    offsets, slots, places = g.group_by_expert(experts, layer.gate_up_q.shape[0], layer.first_expert)
    x_q, x_scale = g.quantize_per_token(x)
    h = g.matmul_experts_swiglu(x_q, layer.gate_up_q, x_scale, layer.gate_up_scale, offsets, slots, k)
    h_q, h_scale = g.quantize_per_token(h)
    y = g.matmul_experts(h_q, layer.down_q, h_scale, layer.down_scale, offsets)
    return g.combine_experts(y, weights, places, add)


@pytest.mark.parametrize("T", [1, 2, 17, 130, 600])
@pytest.mark.parametrize("E,H,inner,k", [(4, 64, 48, 2), (16, 272, 144, 4), (64, 256, 128, 8)])
def test_layer_is_its_steps(T, E, H, inner, k):
    router = dict(scoring="sigmoid", bias=torch.randn(E) * 0.1, groups=4, top_groups=3, group_score="top2" if E > 4 else "max", scale=2.5) if E >= 16 else {}
    layer, gen = _layer(E, H, inner, k, seed=T, **router)
    layer = layer.cuda()
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(T, H, generator=gen).to(dtype).cuda()
        logits = torch.randn(T, E, generator=gen).to(dtype).cuda()
        add = torch.randn(T, H, generator=gen).to(torch.bfloat16).cuda()
        assert torch.equal(layer(x, logits), _step_by_step(layer, x, logits))
        assert torch.equal(layer(x, logits, add), _step_by_step(layer, x, logits, add))


def test_layer_against_float_weights():
    """W8A8 with per-token and per-channel scales keeps an experts' block to about one per cent in the 2-norm: two quantised products, each with
    two operands whose rounding errors are uniform with a 1/sqrt(12) step of 1/127 of a row's largest value (about 3 sigma of 256 Gaussians:
    3 / 127 / 3.46 = 0.7 % of sigma per operand), add up to 0.7 % * sqrt(4) = 1.4 % and the bf16 rounding."""
    layer, gen = _layer(16, 256, 256, 4, seed=1)
    x, logits = torch.randn(64, 256, generator=gen), torch.randn(64, 16, generator=gen)
    gen2 = torch.Generator().manual_seed(1)
    gate_up = torch.randn(16, 512, 256, generator=gen2) * 256 ** -0.5
    down = torch.randn(16, 256, 256, generator=gen2) * 256 ** -0.5
    w, e = R.route(logits, 4)
    exact = torch.zeros(64, 256, dtype=torch.float64)
    for t in range(64):
        for j in range(4):
            i = int(e[t, j])
            _, h = R.swiglu(x[t].double()[None] @ gate_up[i].double().t())
            exact[t] += w[t, j] * (h @ down[i].double().t())[0]
    out = layer.cuda()(x.cuda(), logits.cuda()).cpu().double()
    assert (out - exact).norm() <= 0.025 * exact.norm()


def test_ranks_add_up():
    """Two modules that hold half of the experts each, the second on top of the first, against one that holds all."""
    import gemm_int8_b200 as g

    layer, gen = _layer(16, 128, 64, 4, seed=3)
    x, logits = torch.randn(40, 128, generator=gen).cuda(), torch.randn(40, 16, generator=gen).cuda()
    whole = layer.cuda()(x, logits).double()
    halves = [g.Int8Experts(layer.gate_up_q[a:a + 8], layer.gate_up_scale[a:a + 8], layer.down_q[a:a + 8], layer.down_scale[a:a + 8], 4, first_expert=a) for a in (0, 8)]
    parts = [h(x, logits) for h in halves]
    # each half is rounded to bf16 once more than its share of the whole
    bound = 2 ** -8 * (whole.abs() + parts[0].double().abs() + parts[1].double().abs()) + 1e-6
    assert ((parts[0].double() + parts[1].double() - whole).abs() <= bound).all()


def test_masked_tokens_and_odd_shapes():
    layer, gen = _layer(8, 64, 32, 2, seed=5)
    layer = layer.cuda()
    x = torch.randn(2, 3, 64, generator=gen).cuda()
    logits = torch.randn(2, 3, 8, generator=gen).cuda()
    logits[1, 2] = float("-inf")     # this token goes nowhere
    logits[0, 1, 1:] = float("-inf")  # this one to one expert
    add = torch.randn(2, 3, 64, generator=gen).cuda()
    out = layer(x, logits, add)
    assert out.shape == x.shape and torch.equal(out[1, 2], add[1, 2].to(torch.bfloat16))
    assert torch.equal(layer(x.half(), logits.half(), add), layer(x.half().bfloat16(), logits.half().float(), add))
    assert layer(x[:0], logits[:0]).shape == (0, 3, 64)


def test_graph_replays_with_other_tokens():
    """Captured once, replayed with logits that send other numbers of rows to the experts, next to eager calls on another stream."""
    layer, gen = _layer(16, 256, 128, 4, seed=7)
    layer = layer.cuda()
    batches = [(torch.randn(48, 256, generator=gen).cuda(), torch.randn(48, 16, generator=gen).cuda() * s) for s in (1.0, 5.0, 0.0)]
    expected = [layer(x, l) for x, l in batches]
    x_in, l_in = (t.clone() for t in batches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x_in, l_in)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x_in, l_in)
        graphs.append((graph, out))
    for (x, l), want in zip(batches, expected):
        x_in.copy_(x), l_in.copy_(l)
        for graph, out in graphs:
            graph.replay()
            with torch.cuda.stream(side):
                eager = layer(x, l)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(eager, want)


def test_compiles_whole():
    layer, gen = _layer(8, 64, 32, 2, seed=9)
    layer = layer.cuda()
    x, logits = torch.randn(5, 64, generator=gen).cuda(), torch.randn(5, 8, generator=gen).cuda()
    compiled = torch.compile(layer, fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(x, logits), layer(x, logits))
