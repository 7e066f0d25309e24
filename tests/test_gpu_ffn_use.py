"""The operators as they are used: a feed-forward block in either 8-bit type, captured and replayed, on streams, two at once, in place through the C ABI."""
import ctypes

import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu
F8 = R.F8


class _Block:
    """norm -> gate and up product -> SwiGLU -> down product, the sum of the residual stream in the next norm."""

    def __init__(self, H, I, dtype, seed=0):
        from gemm_int8_b200 import quant

        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.norm = dtype, (1 + 0.1 * torch.randn(H, generator=gen, device="cuda")).bfloat16()
        self.w = [torch.randn(2 * I, H, generator=gen, device="cuda") * 0.03, torch.randn(H, I, generator=gen, device="cuda") * 0.03]
        self.q = [quant.quantize_weight_block(w, dtype=dtype) for w in self.w]

    def __call__(self, x, stream):
        import gemm_int8_b200 as g

        mm = g.matmul_blockwise_fp8 if self.dtype == F8 else g.matmul_blockwise
        q, s, stream = g.rms_norm_quantize(x, self.norm, stream, 1e-5, dtype=self.dtype)
        gate_up = mm(q, self.q[0][0], s, self.q[0][1])
        q, s = g.swiglu_quantize(gate_up, dtype=self.dtype)
        return mm(q, self.q[1][0], s, self.q[1][1]), stream

    def exact(self, x, stream):
        v, h = R.norm(x, self.norm, stream, 1e-5)
        gate, up = (v @ self.w[0].double().t()).chunk(2, 1)
        return (gate * torch.sigmoid(gate) * up) @ self.w[1].double().t(), h


@pytest.mark.parametrize("dtype", [torch.int8, F8])
@pytest.mark.parametrize("M,H,I", [(1, 1024, 1408), (16, 512, 2048), (77, 1040, 2832), (600, 2048, 1408)])
def test_block(M, H, I, dtype):
    """Against the block in 64 bits with the weights before their quantisation.  Errors of independent roundings: activations and weights of either product are off by the rms of
    their quantisation (int8: a step of amax/127 uniform, about 3.5/127/sqrt(12) = 0.8 %; e4m3: 2.6 %), so a product by sqrt(2) times that, the SwiGLU (two
    factors, one with a slope up to 1.1) by 1.5 times that again, the down product adds its own: below 3.2 times 0.8 % and 2.6 %; twice that is allowed."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(M)
    block = _Block(H, I, dtype)
    x = torch.randn(M, H, generator=gen, device="cuda").bfloat16()
    stream = torch.randn(M, H, generator=gen, device="cuda").bfloat16()
    out, total = block(x, stream)
    want, h = block.exact(x, stream)
    assert torch.equal(total, h.float().bfloat16())
    rel = float((out.double() - want).norm() / want.norm())
    assert rel < 2 * 3.2 * (0.008 if dtype == torch.int8 else 0.026), rel
    g.check_device()


@pytest.mark.parametrize("dtype", [torch.int8, F8])
def test_captured_block_replays_with_other_tokens(dtype):
    block = _Block(512, 768, dtype)
    x, stream = torch.zeros(24, 512, dtype=torch.bfloat16, device="cuda"), torch.zeros(24, 512, dtype=torch.float32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x, stream)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same layer
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(block(x, stream))
        graphs.append(graph)
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(24, 512, generator=gen, device="cuda"))
        stream.copy_(torch.randn(24, 512, generator=gen, device="cuda"))
        for graph in graphs:
            graph.replay()
        want = block(x.clone(), stream.clone())
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_streams_and_calls_at_once():
    """Calls on two streams at once give what they give one after the other."""
    import gemm_int8_b200 as g

    blocks = [_Block(1024, 1408, d, seed=i) for i, d in enumerate((torch.int8, F8))]
    data = [(R.outliers(torch.Generator(device="cuda").manual_seed(i), 300, 1024, torch.bfloat16), torch.randn(300, 1024, device="cuda")) for i in range(2)]
    want = [b(*d) for b, d in zip(blocks, data)]
    streams = [torch.cuda.Stream() for _ in blocks]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(blocks[i](*data[i]))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        for o in many:
            assert all(torch.equal(a, b) for a, b in zip(o, w))
    g.check_device()


def test_one_call_right_behind_the_other():
    """Each operator is a programmatic dependent of the one in front: what it reads has been written, what it writes is read no more."""
    import gemm_int8_b200 as g

    block = _Block(512, 640, F8)
    x, stream = torch.randn(9, 512, device="cuda").bfloat16(), torch.randn(9, 512, device="cuda").bfloat16()

    def run(sync):
        y, s = x, stream
        for _ in range(40):
            y, s = block(y, s)
            if sync:
                torch.cuda.synchronize()
        return y, s

    a, b = run(True), run(False)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g.check_device()


@pytest.mark.parametrize("M,N,K", [(4, 2048, 2048), (16, 4096, 512), (40, 1024, 4096), (150, 600, 1040), (600, 4096, 512)])
def test_weights_written_right_in_front_of_the_layer(M, N, K):
    """The product requests weights while the layer's quantiser still runs: they were written before that was let start, by the copy in front."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(N)
    layers = [g.Fp8Linear.from_float(torch.randn(N, K, generator=gen, device="cuda") * 0.03) for _ in range(2)]
    x = torch.randn(M, K, generator=gen, device="cuda").bfloat16()
    want = [layer(x) for layer in layers]
    changing = g.Fp8Linear(layers[0].weight_q.clone(), layers[0].weight_scale.clone())
    torch.cuda.synchronize()
    got = []
    for i in range(20):
        changing.weight_q.view(torch.uint8).copy_(layers[i % 2].weight_q.view(torch.uint8))
        changing.weight_scale.copy_(layers[i % 2].weight_scale)
        got.append(changing(x))
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2]), i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_total_in_place(dtype):
    """The C entry may write the sum over the residual, or over x of the same type."""
    import gemm_int8_b200 as g

    M, H = 300, 4096
    x, r, w = torch.randn(M, H, device="cuda").to(dtype), torch.randn(M, H, device="cuda").to(dtype), torch.randn(H, device="cuda")
    want = g.rms_norm_quantize(x, w, r)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for onto_x in (False, True):
        a, b = x.clone(), r.clone()
        q, s = torch.empty(M, H, dtype=torch.int8, device="cuda"), torch.empty(M, H // 128, device="cuda")
        total = a if onto_x else b
        code = 0 if dtype == torch.float32 else 1
        assert g._C.gi8_rms_norm_quantize(p(a), code, p(b), code, p(w), 0, 1e-6, p(total), p(q), 0, p(s), 1, M, H, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        assert torch.equal(q, want[0]) and torch.equal(s, want[1]) and torch.equal(total, want[2])


def test_nothing_behind_the_results_is_touched():
    """Through the C ABI into the middle of larger buffers: the bytes around q, scales, total and out stay."""
    import gemm_int8_b200 as g

    M, H, N = 5, 1040, 200
    KB = 9
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    x, w = torch.randn(M, H, device="cuda").bfloat16(), torch.randn(H, device="cuda").bfloat16()
    p = lambda t, at: ctypes.c_void_p(t.data_ptr() + at)  # noqa: E731
    for q_type in (0, 1):
        q, s, t = (torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") for n in (M * H + 64, M * KB * 4 + 64, M * H * 2 + 64))
        assert g._C.gi8_rms_norm_quantize(p(x, 0), 1, p(x, 0), 1, p(w, 0), 1, 1e-6, p(t, 32), p(q, 32), q_type, p(s, 32), 1, M, H, stream) == 0
        for b in (q, s, t):
            assert bool((b[:32] == 0x5A).all()) and bool((b[-32:] == 0x5A).all())
        q, s = (torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") for n in (M * (H // 2 - 8) + 64, M * 4 * 5 + 64))
        assert g._C.gi8_swiglu_quantize(p(x[:, : H - 16].contiguous(), 0), 1, p(q, 32), q_type, p(s, 32), 1, M, H // 2 - 8, stream) == 0
        for b in (q, s):
            assert bool((b[:32] == 0x5A).all()) and bool((b[-32:] == 0x5A).all())
    x_q, w_q = torch.randn(M, H, device="cuda").to(F8), torch.randn(N, H, device="cuda").to(F8)
    sx, sw = torch.rand(M, KB, device="cuda"), torch.rand(2, KB, device="cuda")
    for rows in (M, 1):
        out = torch.full((rows * N * 2 + 64,), 0x5A, dtype=torch.uint8, device="cuda")
        assert g._C.gi8_fp8_matmul_blockwise(p(x_q, 0), p(w_q, 0), p(sx, 0), KB, p(sw, 0), KB, p(out, 32), rows, N, H, stream) == 0
        assert bool((out[:32] == 0x5A).all()) and bool((out[-32:] == 0x5A).all())


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: the last rows are what they are by themselves."""
    import gemm_int8_b200 as g

    def same(many, few, rows):
        for a, b in zip(many, few):
            assert torch.equal(a[-rows:].contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))

    M, H = 132000, 16400
    x, w = torch.empty(M, H, dtype=torch.bfloat16, device="cuda"), torch.ones(H, device="cuda")
    x.view(torch.int16).copy_((torch.arange(M * 16, device="cuda", dtype=torch.int32).reshape(M, 16) % 16000).to(torch.int16).repeat(1, H // 16))
    for kw in ({"dtype": F8}, {"scales": "token"}):
        same(g.rms_norm_quantize(x, w, x, **kw), g.rms_norm_quantize(x[-300:], w, x[-300:], **kw), 300)
        same(g.swiglu_quantize(x[:, :16384], **kw), g.swiglu_quantize(x[-300:, :16384], **kw), 300)
    same(g.quantize_per_token_block(x, F8), g.quantize_per_token_block(x[-300:], F8), 300)
    del x
    M, N, K = 66000, 32784, 256
    gen = torch.Generator(device="cuda").manual_seed(0)
    x_q, w_q = (torch.randint(-7, 8, (r, K), generator=gen, device="cuda").to(F8) for r in (M, N))
    sx, sw = torch.ones(M, 2, device="cuda"), torch.ones(-(-N // 128), 2, device="cuda")
    out = g.matmul_blockwise_fp8(x_q, w_q, sx, sw)
    assert torch.equal(out[-500:], (x_q[-500:].double() @ w_q.double().t()).float().bfloat16())
    g.check_device()


def test_opcheck_and_compile():
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(3)
    ops = torch.ops.gemm_int8_CUDA
    x, residual, weight = torch.randn(5, 272, generator=gen, device="cuda").bfloat16(), torch.randn(5, 272, generator=gen, device="cuda"), torch.ones(272, device="cuda")
    q, s = g.quantize_per_token_block(x, F8)
    layer = g.Fp8Linear.from_float(torch.randn(544, 272, generator=gen, device="cuda"), torch.randn(544, generator=gen, device="cuda"))
    every = ("test_schema", "test_autograd_registration", "test_faketensor")
    for blockwise, e4m3 in ((True, True), (True, False), (False, False)):
        checks = every[e4m3:]  # (the check of the schema multiplies what comes back, which torch cannot do in 8-bit floating point)
        torch.library.opcheck(ops.rms_norm_quantize.default, (x, weight, residual, 1e-6, blockwise, e4m3), test_utils=checks)
        torch.library.opcheck(ops.rms_norm_quantize.default, (x, weight, None, 1e-6, blockwise, e4m3), test_utils=checks)
        torch.library.opcheck(ops.swiglu_quantize.default, (x[:, :256], blockwise, e4m3), test_utils=checks)
    checks = every[1:]
    torch.library.opcheck(ops.fp8_quantize_token_block.default, (x,), test_utils=checks)
    torch.library.opcheck(ops.fp8_matmul_blockwise.default, (q, layer.weight_q, s, layer.weight_scale), test_utils=checks)
    for bias in (layer.bias, None):
        torch.library.opcheck(ops.fp8_linear.default, (x, layer.weight_q, layer.weight_scale, bias), test_utils=checks)

    def block(x, residual):
        q, s, total = g.rms_norm_quantize(x, weight, residual, dtype=F8)
        gate_up = g.matmul_blockwise_fp8(q, layer.weight_q, s, layer.weight_scale)
        return (*g.swiglu_quantize(gate_up, dtype=F8), total, layer(x))

    compiled = torch.compile(block, fullgraph=True, backend="aot_eager")
    for rows in (5, 1, 3):
        for a, b in zip(compiled(x[:rows], residual[:rows]), block(x[:rows], residual[:rows])):
            assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
