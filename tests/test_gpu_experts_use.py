"""The experts' operators as programs use them: on other streams, captured, two calls at once, behind one another, the same buffers again."""
import pytest
import torch

import experts_reference as R

pytestmark = pytest.mark.gpu


def _state(T, E, k, H, inner, seed):
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(seed)
    gate_up = torch.randn(E, 2 * inner, H, generator=gen) * H ** -0.5
    down = torch.randn(E, H, inner, generator=gen) * inner ** -0.5
    layer = g.Int8Experts.from_float(gate_up.cuda(), down.cuda(), k)
    return layer, torch.randn(T, H, generator=gen).bfloat16().cuda(), torch.randn(T, E, generator=gen).cuda()


def test_two_streams_at_once():
    """Calls of different sizes on two streams, many in flight: nothing is shared between them."""
    states = [_state(*a) for a in ((3, 8, 2, 128, 64, 1), (300, 16, 4, 256, 128, 2))]
    want = [layer(x, l) for layer, x, l in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for _ in range(30):
        for i, (layer, x, l) in enumerate(states):
            with torch.cuda.stream(streams[i]):
                got[i].append(layer(x, l))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_each_step_sees_the_one_in_front():
    """A chain of every operator, tens of times over without a wait in between, on inputs that change from pass to pass and in buffers that are
    used again (the allocator hands the freed ones out)."""
    import gemm_int8_b200 as g

    layer, x, logits = _state(200, 16, 4, 256, 128, 3)
    inputs = [(x.roll(i, 0), logits.roll(i, 0)) for i in range(6)]
    want = [layer(a, b) for a, b in inputs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for a, b in inputs:
            w, e = g.route_experts(b, 4)
            offsets, slots, places = g.group_by_expert(e, 16)
            a_q, a_s = g.quantize_per_token(a)
            h = g.matmul_experts_swiglu(a_q, layer.gate_up_q, a_s, layer.gate_up_scale, offsets, slots, 4)
            h_q, h_s = g.quantize_per_token(h)
            got.append(g.combine_experts(g.matmul_experts(h_q, layer.down_q, h_s, layer.down_scale, offsets), w, places))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_weights_written_right_in_front():
    """The weights and scales of a call may be the work of the launch directly in front of it."""
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(4)
    x_q = torch.randint(-128, 128, (40, 512), dtype=torch.int8, generator=gen)
    ws = [torch.randint(-128, 128, (6, 256, 512), dtype=torch.int8, generator=gen) for _ in range(4)]
    sx, sw = torch.rand(40, generator=gen), torch.rand(6, 256, generator=gen)
    offsets = torch.tensor([0, 3, 3, 20, 21, 30, 40], dtype=torch.int32)
    want = [R.product(x_q, w, sx, sw, offsets)[1].to(torch.bfloat16) for w in ws]
    x_d, sx_d, sw_d, off_d = x_q.cuda(), sx.cuda(), sw.cuda(), offsets.cuda()
    ws = [w.cuda() for w in ws]
    buf = torch.empty_like(ws[0])
    for _ in range(3):
        got = []
        for w in ws:
            buf.copy_(w)
            got.append(g.matmul_experts(x_d, buf, sx_d, sw_d, off_d))
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_offsets_written_right_in_front_of_a_captured_product():
    import gemm_int8_b200 as g

    gen = torch.Generator().manual_seed(5)
    x_q = torch.randint(-128, 128, (64, 256), dtype=torch.int8, generator=gen)
    w = torch.randint(-128, 128, (4, 128, 256), dtype=torch.int8, generator=gen)
    sx, sw = torch.rand(64, generator=gen), torch.rand(4, 128, generator=gen)
    all_offsets = [torch.tensor(o, dtype=torch.int32) for o in ([0, 16, 32, 48, 64], [0, 0, 0, 0, 64], [0, 64, 64, 64, 64], [0, 1, 2, 3, 4], [0, 0, 0, 0, 0])]
    x_d, w_d, sx_d, sw_d = x_q.cuda(), w.cuda(), sx.cuda(), sw.cuda()
    source, off = all_offsets[0].cuda(), all_offsets[0].cuda()
    g.matmul_experts(x_d, w_d, sx_d, sw_d, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        off.copy_(source)
        out = g.matmul_experts(x_d, w_d, sx_d, sw_d, off)
    for o in all_offsets:
        source.copy_(o)
        graph.replay()
        assert torch.equal(out.cpu(), R.product(x_q, w, sx, sw, o)[1].to(torch.bfloat16))


def test_one_token_to_the_same_expert_twice():
    """A token that names an expert more often than once has a row for each, and more rows than tokens go to an expert."""
    import gemm_int8_b200 as g

    experts = torch.tensor([[2, 2, 2, 0]], dtype=torch.int32).repeat(40, 1)
    offsets, slots, places = g.group_by_expert(experts.cuda(), 3)
    assert offsets.tolist() == [0, 40, 40, 160]
    gen = torch.Generator().manual_seed(6)
    x_q = torch.randint(-128, 128, (40, 128), dtype=torch.int8, generator=gen)
    w = torch.randint(-128, 128, (3, 64, 128), dtype=torch.int8, generator=gen)
    sx, sw = torch.rand(40, generator=gen), torch.rand(3, 64, generator=gen)
    out = g.matmul_experts(x_q.cuda(), w.cuda(), sx.cuda(), sw.cuda(), offsets, slots, 4)
    _, single = R.product(x_q, w, sx, sw, offsets.cpu(), slots.cpu(), 4)
    assert torch.equal(out.cpu(), single.to(torch.bfloat16))


def test_results_do_not_depend_on_the_batch():
    """A token's result is the same alone and in a batch (integer sums, and no atomics anywhere)."""
    layer, x, logits = _state(130, 8, 2, 256, 128, 7)
    whole = layer(x, logits)
    for t in (0, 64, 129):
        assert torch.equal(layer(x[t:t + 1], logits[t:t + 1])[0], whole[t])


def test_results_beyond_32_bits():
    """Rows whose offset in the result passes 2^31 elements."""
    import gemm_int8_b200 as g

    rows, N, K = 140000, 16384, 16
    if torch.cuda.mem_get_info()[0] < 20e9:
        pytest.skip("needs 20 GB")
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randint(-128, 128, (rows, K), dtype=torch.int8, device="cuda", generator=gen)
    w = torch.randint(-128, 128, (2, N, K), dtype=torch.int8, device="cuda", generator=gen)
    sx, sw = torch.rand(rows, device="cuda", generator=gen), torch.rand(2, N, device="cuda", generator=gen)
    offsets = torch.tensor([0, 70001, 139990], dtype=torch.int32, device="cuda")
    out = g.matmul_experts(x, w, sx, sw, offsets)
    for a, b, e in ((0, 300, 0), (69900, 70001, 0), (70001, 70100, 1), (139700, 139990, 1)):
        acc = (x[a:b].double() @ w[e].double().t()).float()
        assert torch.equal(out[a:b], (acc * (sx[a:b, None] * sw[e][None])).bfloat16())
    assert (out[139990:] == 0).all()
    places = torch.tensor([[139989, 5], [139000, -1]], dtype=torch.int32, device="cuda")
    s = g.combine_experts(out, torch.ones(2, 2, device="cuda"), places)
    assert torch.equal(s[1], out[139000]) and torch.equal(s[0], (out[139989].float() + out[5].float()).bfloat16())


def test_ordinary_launches_give_the_same(monkeypatch):
    """GEMM_INT8_PDL=0: every launch waits for the one in front as a whole, and no weight is requested early."""
    import gemm_int8_b200 as g

    states = [_state(*a, seed) for seed, a in enumerate(((1, 8, 2, 128, 64), (40, 16, 4, 256, 128), (700, 4, 2, 256, 192)))]
    want = [layer(x, l) for layer, x, l in states]
    try:
        monkeypatch.setenv("GEMM_INT8_PDL", "0")
        g.reload_env()
        assert all(torch.equal(layer(x, l), w) for (layer, x, l), w in zip(states, want))
    finally:
        monkeypatch.delenv("GEMM_INT8_PDL")
        g.reload_env()
    assert all(torch.equal(layer(x, l), w) for (layer, x, l), w in zip(states, want))


def test_each_pass_of_a_layer_waits_for_its_weights():
    """The layer requests its first weights early: weights that change between two calls are those of the call."""
    import gemm_int8_b200 as g

    layer, x, logits = _state(24, 8, 2, 512, 256, 9)
    other, _, _ = _state(24, 8, 2, 512, 256, 10)
    want = [layer(x, logits), other(x, logits)]
    versions = [tuple(getattr(m, n).clone() for n in ("gate_up_q", "gate_up_scale", "down_q", "down_scale")) for m in (layer, other)]
    got = []
    for i in range(20):
        for n, v in zip(("gate_up_q", "gate_up_scale", "down_q", "down_scale"), versions[i % 2]):
            getattr(layer, n).copy_(v)
        got.append(layer(x, logits))
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(got))
    assert g.device_status() == 0
