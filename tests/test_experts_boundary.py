"""What the experts' operators refuse, before any device is touched, and their fake kernels."""
import ctypes
import os

import pytest
import torch

import test_kernel_waits as W


@pytest.fixture
def call():
    import gemm_int8_b200 as g

    buf = ctypes.create_string_buffer(8192 + 256)
    base = (ctypes.addressof(buf) + 255) & ~255
    C = g._C
    C._keep = buf

    def f(name, **over):
        p = {"p": base}
        p.update(over)
        a = ctypes.c_void_p

        def arg(k, default):
            return over[k] if k in over else default

        if name == "route":
            return C.gi8_route_experts(a(arg("logits", base)), arg("dtype", 0), a(arg("bias", None)), a(arg("weights", base)), a(arg("experts", base)), arg("T", 4), arg("E", 16),
                                       arg("k", 2), 0, arg("groups", 1), arg("top_groups", 1), 0, 1, 1.0, None)
        if name == "group":
            return C.gi8_group_by_expert(a(arg("experts", base)), arg("S", 8), arg("E", 4), arg("first", 0), a(arg("offsets", base)), a(arg("slots", base)), a(arg("places", base)), a(arg("ws", None)), arg("ws_bytes", 0), None)
        if name == "product":
            return C.gi8_matmul_experts(a(arg("x", base)), a(arg("w", base)), a(arg("sx", base)), a(arg("sw", base)), a(arg("offsets", base)), a(arg("slots", None)), arg("k", 1),
                                        a(arg("out", base)), arg("rows", 8), arg("tokens", 8), arg("E", 2), arg("N", 16), arg("K", 32), arg("swiglu", 0), None)
        if name == "combine":
            return C.gi8_combine_experts(a(arg("y", base)), a(arg("weights", base)), a(arg("places", base)), a(arg("add", None)), a(arg("out", base)), arg("T", 4), arg("k", 2),
                                         arg("rows", 8), arg("N", 16), None)
        return C.gi8_experts(a(arg("x", base)), arg("x_dtype", 1), a(arg("logits", base)), arg("logits_dtype", 0), a(arg("bias", None)), a(arg("gate_up", base)), a(base), a(base), a(base),
                             a(arg("add", None)), a(arg("out", base)), a(arg("scratch", base)), arg("bytes", 1 << 30), arg("T", 4), arg("H", 64), arg("I", 32), arg("ER", 8), arg("E", 8),
                             arg("first", 0), arg("k", 2), 0, arg("groups", 1), arg("top_groups", 1), 0, 1, 1.0, None)

    f.base, f.C = base, C
    return f


def test_router_refuses(call):
    assert call("route", E=0) == 2 and call("route", E=1025) == 2
    assert call("route", k=0) == 2 and call("route", k=33, E=64) == 2 and call("route", k=17) == 2
    assert call("route", groups=3) == 2 and call("route", groups=0) == 2 and call("route", groups=64, E=128) == 2
    assert call("route", groups=4, top_groups=5) == 2 and call("route", groups=4, top_groups=0) == 2
    assert call("route", groups=8, top_groups=1, k=3) == 2  # one group of two cannot hold three
    assert call("route", dtype=2) == 1 and call("route", T=-1) == 1 and call("route", logits=None) == 1
    assert call("route", logits=call.base + 2) == 3 and call("route", dtype=1, logits=call.base + 1) == 3 and call("route", bias=call.base + 2) == 3
    assert call("route", T=0, logits=None) == 0


def test_grouping_refuses(call):
    assert call("group", E=0) == 2 and call("group", E=1025) == 2 and call("group", S=-1) == 2 and call("group", S=(1 << 24) + 1) == 2
    assert call("group", first=-1) == 1 and call("group", first=2 ** 31 - 2) == 1
    assert call("group", offsets=None) == 1 and call("group", slots=None) == 1 and call("group", places=call.base + 2) == 3
    need = call.C.gi8_group_by_expert_workspace_bytes(8193, 4)
    assert need > 0 and call.C.gi8_group_by_expert_workspace_bytes(8192, 4) == 0
    assert call("group", S=8193) == 6 and call("group", S=8193, ws=call.base, ws_bytes=need - 1) == 6 and call("group", S=8193, ws=call.base + 2, ws_bytes=need) == 3


def test_product_refuses(call):
    assert call("product", K=24) == 2 and b"multiple of 16" in call.C.gi8_last_error()
    assert call("product", K=131072) == 2 and call("product", E=0) == 2 and call("product", E=1025) == 2
    assert call("product", rows=-1) == 1 and call("product", tokens=7) == 1 and call("product", k=0) == 1
    assert call("product", N=1 << 30, E=2) == 2 and call("product", N=1 << 29, E=2, swiglu=1) == 2
    assert call("product", x=call.base + 8) == 3 and call("product", w=None) == 1 and call("product", out=call.base + 1) == 3
    assert call("product", sx=None) == 1 and call("product", offsets=None) == 1 and call("product", slots=call.base + 2) == 3
    assert call("product", rows=0) == 0 and call("product", N=0) == 0


def test_sum_refuses(call):
    assert call("combine", k=0) == 2 and call("combine", k=33) == 2 and call("combine", T=-1) == 1
    assert call("combine", y=None) == 1 and call("combine", out=call.base + 1) == 3 and call("combine", weights=call.base + 2) == 3
    assert call("combine", T=0) == 0 and call("combine", N=0) == 0


def test_layer_refuses_before_it_launches(call):
    """Without a device the first launch fails with GI8_ERR_CUDA, so any other status was given in front of it."""
    assert call("layer", H=72) == 2 and call("layer", I=40) == 2 and call("layer", I=0) == 2 and call("layer", H=131072) == 2
    assert call("layer", E=9) == 1 and call("layer", first=1) == 1 and call("layer", first=-1) == 1
    assert call("layer", k=9) == 2 and call("layer", groups=3) == 2 and call("layer", x_dtype=2) == 1 and call("layer", logits_dtype=3) == 1
    assert call("layer", bytes=1024) == 6 and call("layer", scratch=None) == 1 and call("layer", scratch=call.base + 16) == 3
    assert call("layer", x=call.base + 8) == 3 and call("layer", out=call.base + 1) == 3 and call("layer", add=call.base + 1) == 3
    assert call("layer", T=1 << 28) == 2 and call("layer", T=0) == 0
    n = call.C.gi8_experts_scratch_bytes(4, 64, 32, 8, 2)
    assert n > 0 and n % 256 == 0 and call.C.gi8_experts_scratch_bytes(-1, 64, 32, 8, 2) == 0


def test_python_arguments():
    import gemm_int8_b200 as g

    x = torch.zeros(2, 4)
    with pytest.raises(ValueError):
        g.route_experts(x, 1, scoring="relu")
    with pytest.raises(ValueError):
        g.route_experts(x, 1, group_score="mean")
    for f in (lambda: g.route_experts(x, 1), lambda: g.group_by_expert(x.int(), 4), lambda: g.combine_experts(x.bfloat16(), x, x.int())):
        with pytest.raises((NotImplementedError, RuntimeError)):  # there is no CPU path
            f()


def test_fake_kernels_propagate_shapes():
    import gemm_int8_b200 as g
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        logits = torch.empty(5, 16, device="cuda")
        w, e = g.route_experts(logits, 3)
        assert w.shape == (5, 3) and w.dtype == torch.float32 and e.dtype == torch.int32
        offsets, slots, places = g.group_by_expert(e, 16)
        assert offsets.shape == (17,) and slots.shape == (15,) and places.shape == (5, 3)
        x, wq = torch.empty(5, 32, dtype=torch.int8, device="cuda"), torch.empty(16, 48, 32, dtype=torch.int8, device="cuda")
        sx, sw = torch.empty(5, device="cuda"), torch.empty(16, 48, device="cuda")
        assert g.matmul_experts(x, wq, sx, sw, offsets, slots, 3).shape == (15, 48)
        y = g.matmul_experts_swiglu(x, wq, sx, sw, offsets, slots, 3)
        assert y.shape == (15, 24) and y.dtype == torch.bfloat16
        assert g.combine_experts(y, w, places).shape == (5, 24)
        layer = g.Int8Experts(wq, sw, torch.empty(16, 32, 24, dtype=torch.int8, device="cuda"), torch.empty(16, 32, device="cuda"), 3)
        assert layer(torch.empty(5, 32, device="cuda"), logits).shape == (5, 32)


# The rules on waits that hold for the kernels of the package, read from the sources of these.
_DIR = os.path.join(W.CSRC, "experts")


def _kernels():
    csrc, W.CSRC = W.CSRC, _DIR
    try:
        return W._kernels()
    finally:
        W.CSRC = csrc


def test_all_kernels_are_seen():
    assert {p.id for p in _kernels()} == {"experts_gemm_kernel"}


@pytest.mark.parametrize("body", _kernels())
def test_waits(body):
    W.test_last_commits_are_awaited(body)
    W.test_lanes_of_a_warp_decide_together(body)
    # the named barrier of the epilogue warps is reached by all of them once per tile, whether a wait has failed or not
    loop = body[body.index("asm volatile(\"bar.sync 1, "):]
    assert "break" not in loop[:loop.index("mbar_arrive(&bar_acc_empty")]
