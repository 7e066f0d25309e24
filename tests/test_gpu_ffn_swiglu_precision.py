"""What swiglu_quantize computes before it rounds, to units of fp32 whatever the gate: read from the scales of blocks (or rows) that hold one value."""
import pytest
import torch

from test_gpu_ffn_swiglu_range import FORMS, _rel

pytestmark = pytest.mark.gpu

# Units of 2^-24 of the value: ex2.approx 4 (two units in the last place); fp32: ln 2 in fp32 4 (its rounding, 1.9e-9, times an exponent of at most 115); bf16: the square that the
# correction leaves out 2; 1 - r and 1 + e 2, the reciprocal 2 (one unit in the last place), two products 2, the scale's division 1.
UNITS = 15


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lo,hi,up", [(-1e-3, 1e-3, 1.0), (-8.0, 8.0, 1.0), (-64.0, -8.0, 1.0), (8.0, 200.0, 1.0), (-80.0, -60.0, 1.0), (1e-38, 1e-36, 1e20)])
def test_value_of_one(lo, hi, up, x, scales, dtype):
    gen = torch.Generator(device="cuda").manual_seed(17)
    gates = torch.rand(4096, generator=gen, device="cuda", dtype=torch.float64) * (hi - lo) + lo
    ups = up * (0.5 + 0.5 * torch.rand(4096, generator=gen, device="cuda", dtype=torch.float64))
    rel = _rel(gates.float(), ups.float(), scales, dtype, x)
    assert float(rel.max()) <= UNITS * 2.0 ** -24, (float(rel.max()) * 2 ** 24, float(gates[rel.argmax()]))


@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
def test_value_of_one_in_rows_beyond_the_registers(x):
    """Rows of more than 32768 features with a scale per token are read twice behind the first 32768."""
    gen = torch.Generator(device="cuda").manual_seed(18)
    gates = torch.rand(64, generator=gen, device="cuda") * 72 - 64
    assert float(_rel(gates, torch.ones(64, device="cuda"), "token", torch.int8, x, N=40016).max()) <= UNITS * 2.0 ** -24
