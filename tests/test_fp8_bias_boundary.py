"""What gi8_fp8_linear_bias_f32 refuses before any device is touched."""
import ctypes

import pytest
import torch


@pytest.fixture
def call():
    import gemm_int8_b200 as g

    buf = ctypes.create_string_buffer(8192 + 256)
    base = (ctypes.addressof(buf) + 255) & ~255

    def f(**over):
        _ = buf
        p = lambda k, default=base: ctypes.c_void_p(over.get(k, default))  # noqa: E731
        return g._C.gi8_fp8_linear_bias_f32(p("x"), over.get("x_dtype", 0), p("w"), p("sw"), over.get("ld_w", 1), p("bias"), p("xq"), p("xs"), p("out"), over.get("M", 4),
                                            over.get("N", 8), over.get("K", 64), None)

    f.base = base
    return f


def test_refusals(call):
    b = call.base
    assert call(bias=b + 2) == 3 and call(bias=b + 1) == 3 and call(sw=b + 2) == 3 and call(xq=b + 8) == 3 and call(xs=b + 2) == 3 and call(out=b + 1) == 3
    for k in ("x", "w", "sw", "xq", "xs", "out"):
        assert call(**{k: None}) == 1, k
    assert call(K=24) == 2 and call(K=0) == 2 and call(K=131072) == 2 and call(ld_w=0) == 1 and call(x_dtype=2) == 1 and call(M=-1) == 1
    assert call(M=0) == 0 and call(N=0) == 0 and call(K=0, M=0) == 0
    # what passes the checks meets the missing device, with a bias at any 4-byte address and without one
    if not torch.cuda.is_available():
        assert call() in (4, 5) and call(bias=b + 4) in (4, 5) and call(bias=None) in (4, 5)


def test_layer_keeps_its_bias():
    import gemm_int8_b200 as g

    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        layer = g.Fp8Linear.from_float(torch.randn(16, 32), torch.randn(16).to(dtype))
        assert layer.bias.dtype == dtype
