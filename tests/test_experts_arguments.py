"""Arguments of the experts' operators that are refused, or limited, before any device is touched."""
import pytest
import torch

from test_experts_boundary import call  # noqa: F401  (the fixture)


def test_slots_need_the_number_of_choices():
    """Without it every row would read another token than its own."""
    import gemm_int8_b200 as g
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(5, 32, dtype=torch.int8, device="cuda"), torch.empty(4, 16, 32, dtype=torch.int8, device="cuda")
        sx, sw = torch.empty(5, device="cuda"), torch.empty(4, 16, device="cuda")
        offsets, slots = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(10, dtype=torch.int32, device="cuda")
        for f in (g.matmul_experts, g.matmul_experts_swiglu):
            with pytest.raises(ValueError, match="top_k"):
                f(x, w, sx, sw, offsets, slots)
            assert f(x, w, sx, sw, offsets, slots, 2).shape[0] == 10 and f(x, w, sx, sw, offsets, slots, top_k=2).shape[0] == 10
            assert f(x, w, sx, sw, offsets).shape[0] == 5 and f(x, w, sx, sw, offsets, None, 2).shape[0] == 5


def test_scratch_of_sizes_that_the_layer_refuses(call):
    """0 for whatever the layer refuses by its sizes: 2 T top_k I of the largest arguments is beyond 64 bits."""
    f = call.C.gi8_experts_scratch_bytes
    big = 2 ** 31 - 1
    assert f(big, big, big, 8, 32) == 0
    for T, H, I, E, k in ((big, 64, 32, 8, 2), (2 ** 23 + 1, 64, 32, 8, 2), (4, 131072, 32, 8, 2), (4, 64, 131072, 8, 2), (4, 64, 32, 1025, 2), (4, 64, 32, 8, 33), (4, 64, 32, 0, 2),
                          (4, 0, 32, 8, 2), (4, 64, 0, 8, 2), (4, 64, 32, 8, 0), (2 ** 62, 64, 32, 8, 2)):
        assert f(T, H, I, E, k) == 0, (T, H, I, E, k)
    largest = f(2 ** 19, 131056, 131056, 1024, 32)
    pairs = 2 ** 24
    assert 2 ** 19 * 131056 + pairs * (3 * 131056 + 2 * 131056) < largest < 2 ** 44


def test_first_expert_of_any_size(call):
    """first + E may not wrap around on its way to the comparison with the router's experts."""
    for first in (2 ** 63 - 1, 2 ** 63 - 4, 2 ** 62, 2 ** 31, 1):
        assert call("layer", first=first) == 1, first  # GI8_ERR_INVALID_ARGUMENT
    assert call("layer", first=2 ** 63 - 1, E=1) == 1 and call("layer", first=1, T=0) == 1
    assert call("layer", E=2 ** 62) == 1 and call("layer", E=2 ** 62, first=2 ** 62) == 1
    for first in (2 ** 63 - 1, 2 ** 31):
        assert call("group", first=first) == 1, first


def test_more_tiles_than_are_counted(call):
    """Offsets that do not ascend may give every expert all rows: the products count the tiles of all of them in 32 bits."""
    assert call("product", E=1024, rows=2 ** 28, tokens=2 ** 28) == 2
    assert call("product", E=1024, rows=2 ** 27, tokens=2 ** 27) == 2 and call("product", E=1024, rows=2 ** 27, tokens=4, slots=call.base, k=2) == 2
    assert call("product", E=100, rows=2 ** 31 - 300, tokens=2 ** 31 - 300) == 2


def test_fp32_forms_refuse_as_the_others_do(call, monkeypatch):
    """The C entries whose sum starts from fp32: the checks of the bf16 ones, and alignment to four bytes."""
    C = call.C
    for name, f32 in (("gi8_combine_experts", C.gi8_combine_experts_add_f32), ("gi8_experts", C.gi8_experts_add_f32)):
        monkeypatch.setattr(C, name, f32)
    assert call("combine", k=0) == 2 and call("combine", T=-1) == 1 and call("combine", y=None) == 1 and call("combine", T=0) == 0
    assert call("combine", add=call.base + 2) == 3 and call("combine", out=call.base + 1) == 3
    assert call("layer", H=72) == 2 and call("layer", E=9) == 1 and call("layer", scratch=None) == 1 and call("layer", T=0) == 0
    assert call("layer", add=call.base + 2) == 3
