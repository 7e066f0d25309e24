"""What the operators around the products and the e4m3 product refuse before any device is touched, their fake kernels, and the torch quantisers."""
import ctypes

import pytest
import torch

F8 = torch.float8_e4m3fn


@pytest.fixture
def call():
    import gemm_int8_b200 as g

    buf = ctypes.create_string_buffer(8192 + 256)
    base = (ctypes.addressof(buf) + 255) & ~255
    C, a = g._C, ctypes.c_void_p

    def f(name, **over):
        _ = buf

        def arg(k, default=base):
            v = over.get(k, default)
            return a(v) if isinstance(default, int) and default == base or v is None else v

        if name == "norm":
            return C.gi8_rms_norm_quantize(arg("x"), over.get("x_dtype", 0), arg("residual"), over.get("residual_dtype", 0), arg("weight"), over.get("weight_dtype", 0),
                                           over.get("eps", 1e-6), arg("total"), arg("q"), over.get("q_type", 0), arg("s"), over.get("blocks", 1), over.get("M", 4), over.get("H", 64), None)
        if name == "swiglu":
            return C.gi8_swiglu_quantize(arg("x"), over.get("x_dtype", 0), arg("q"), over.get("q_type", 0), arg("s"), over.get("blocks", 1), over.get("M", 4), over.get("N", 64), None)
        if name == "quantise":
            return C.gi8_fp8_quantize_token_block(arg("x"), over.get("x_dtype", 0), arg("q"), arg("s"), over.get("M", 4), over.get("K", 64), None)
        if name == "product":
            return C.gi8_fp8_matmul_blockwise(arg("x"), arg("w"), arg("sx"), over.get("ld_x", 1), arg("sw"), over.get("ld_w", 1), arg("out"), over.get("M", 4), over.get("N", 8),
                                              over.get("K", 64), None)
        return C.gi8_fp8_linear(arg("x"), over.get("x_dtype", 0), arg("w"), arg("sw"), over.get("ld_w", 1), a(over.get("bias")), arg("xq"), arg("xs"), arg("out"), over.get("M", 4),
                                over.get("N", 8), over.get("K", 64), None)

    f.base, f.C = base, C
    return f


def test_norm_refuses(call):
    b = call.base
    assert call("norm", H=24) == 2 and call("norm", H=32784) == 2 and call("norm", H=131072) == 2 and call("norm", M=1 << 31) == 2
    assert call("norm", M=-1) == 1 and call("norm", H=-16) == 1
    assert call("norm", eps=0.0) == 1 and call("norm", eps=float("nan")) == 1 and call("norm", eps=float("inf")) == 1 and call("norm", eps=-1.0) == 1
    assert call("norm", x_dtype=2) == 1 and call("norm", weight_dtype=-1) == 1 and call("norm", residual_dtype=3) == 1 and call("norm", q_type=2) == 1
    assert call("norm", q_type=1, blocks=0) == 1
    for k in ("x", "weight", "q", "s", "total"):
        assert call("norm", **{k: None}) == 1, k
    for k, by in (("x", 8), ("residual", 8), ("weight", 8), ("total", 8), ("q", 4), ("s", 2)):
        assert call("norm", **{k: b + by}) == 3, k
    assert call("norm", M=0, x=None) == 0 and call("norm", H=0, x=None) == 0
    # what passes the checks meets the missing device
    if not torch.cuda.is_available():
        assert call("norm") in (4, 5) and call("norm", residual=None, total=None) in (4, 5)


def test_swiglu_and_quantiser_refuse(call):
    b = call.base
    assert call("swiglu", N=24) == 2 and call("swiglu", N=131072) == 2 and call("swiglu", M=-1) == 1 and call("swiglu", x_dtype=2) == 1
    assert call("swiglu", q_type=1, blocks=0) == 1 and call("swiglu", q_type=-1) == 1 and call("swiglu", x=None) == 1 and call("swiglu", q=None) == 1
    assert call("swiglu", x=b + 8) == 3 and call("swiglu", q=b + 4) == 3 and call("swiglu", s=b + 2) == 3
    assert call("swiglu", M=0, x=None) == 0
    assert call("quantise", K=12) == 2 and call("quantise", K=4, x_dtype=1) == 2 and call("quantise", x=b + 8) == 3 and call("quantise", q=None) == 1
    assert call("quantise", M=0, x=None) == 0


def test_product_and_linear_refuse(call):
    b = call.base
    assert call("product", K=24) == 2 and call("product", K=131072) == 2 and call("product", M=-1) == 1
    for M in (4, 40):  # either kernel
        assert call("product", M=M, x=None) == 1 and call("product", M=M, sx=None) in (1, 4, 5) and call("product", M=M, x=b + 8) == 3 and call("product", M=M, out=b + 1) == 3
    assert call("product", M=0, x=None) == 0 and call("product", N=0, w=None) == 0
    assert call("linear", sw=None) == 1 and call("linear", sw=b + 2) == 3 and call("linear", bias=b + 1) == 3 and call("linear", xq=b + 8) == 3 and call("linear", xs=b + 2) == 3
    assert call("linear", K=0, bias=b) == 2 and call("linear", K=24) == 2 and call("linear", ld_w=0) == 1 and call("linear", ld_w=1 << 31) == 1
    assert call("linear", M=0) == 0 and call("linear", N=0) == 0 and call("linear", x_dtype=2) == 1


def test_python_arguments():
    import gemm_int8_b200 as g

    x, w = torch.zeros(2, 32), torch.ones(32)
    for f in (lambda **k: g.rms_norm_quantize(x, w, **k), lambda **k: g.swiglu_quantize(x, **k)):
        for kw in ({"scales": "row"}, {"scales": None}, {"dtype": torch.float16}, {"scales": "token", "dtype": F8}):
            with pytest.raises(ValueError):
                f(**kw)
        with pytest.raises((NotImplementedError, RuntimeError)):  # there is no CPU path
            f()
    with pytest.raises(ValueError):
        g.quantize_per_token_block(x, dtype=torch.float16)
    with pytest.raises(ValueError):
        g.Fp8Linear(torch.zeros(16, 16, dtype=torch.int8), torch.ones(1, 1))
    with pytest.raises((NotImplementedError, RuntimeError)):
        g.matmul_blockwise_fp8(x.to(F8), x.to(F8), torch.ones(2, 1), torch.ones(1, 1))


def test_fake_kernels_propagate_shapes():
    import gemm_int8_b200 as g
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(5, 272, device="cuda", dtype=torch.bfloat16), torch.empty(272, device="cuda")
        q, s, t = g.rms_norm_quantize(x, w, torch.empty(5, 272, device="cuda"), dtype=F8)
        assert q.shape == (5, 272) and q.dtype == F8 and s.shape == (5, 3) and t.dtype == torch.float32
        assert len(g.rms_norm_quantize(x, w)) == 2
        q8, s8 = g.swiglu_quantize(torch.empty(5, 544, device="cuda"), scales="token")
        assert q8.shape == (5, 272) and q8.dtype == torch.int8 and s8.shape == (5,)
        assert g.quantize_per_token_block(x, F8)[0].dtype == F8
        out = g.matmul_blockwise_fp8(q, torch.empty(40, 272, device="cuda", dtype=F8), s, torch.empty(1, 3, device="cuda"))
        assert out.shape == (5, 40) and out.dtype == torch.bfloat16
        layer = g.Fp8Linear(torch.empty(40, 272, device="cuda", dtype=F8), torch.empty(1, 3, device="cuda"), torch.empty(40, device="cuda"))
        assert layer(torch.empty(2, 5, 272, device="cuda")).shape == (2, 5, 40)


def test_torch_quantisers_in_e4m3():
    from gemm_int8_b200 import quant

    gen = torch.Generator().manual_seed(0)
    a = torch.randn(200, 300, generator=gen)
    a[3, :128] = 0
    for q, s, rows in ((*quant.quantize_per_token_block(a, dtype=F8), 1), (*quant.quantize_weight_block(a, dtype=F8), 128)):
        assert q.dtype == F8 and q.shape == a.shape and s.shape == (-(-200 // rows), 3)
        back = quant.dequantize_blockwise(q, s, rows)
        # half a step of e4m3: 2^-4 of the value, or half of the smallest number (2^-10) in units of the scale
        unit = s.repeat_interleave(rows, 0)[:200].repeat_interleave(128, 1)[:, :300]
        assert bool(((back - a).abs() <= torch.maximum(a.abs() * 2 ** -4, unit * 2 ** -10) * (1 + 2 ** -20)).all())
    q, s = quant.quantize_per_token_block(a, dtype=F8)
    assert float(s[3, 0]) == 1.0 and not q[3, :128].float().any()
    with pytest.raises(ValueError):
        quant.quantize_weight_block(a, dtype=torch.float16)


# The rules on waits that hold for the kernels of the package, read from the source of the e4m3 product.
def _kernels():
    import os

    import test_kernel_waits as W

    csrc, W.CSRC = W.CSRC, os.path.join(W.CSRC, "fp8")
    try:
        return W._kernels()
    finally:
        W.CSRC = csrc


def test_waits_of_the_e4m3_product():
    import test_kernel_waits as W

    kernels = _kernels()
    assert {p.id for p in kernels} == {"fp8_gemm_kernel"}
    W.test_last_commits_are_awaited(kernels[0].values[0])
    W.test_lanes_of_a_warp_decide_together(kernels[0].values[0])
    # copies that the warps issue themselves have landed before the CTA ends
    body = kernels[0].values[0]
    assert body.rindex("cp_async_wait_all()") > body.rindex("cp_async_arrive(")
