"""Arguments of the experts' operators that are refused, or limited, before any device is touched."""
import pytest
import torch


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
