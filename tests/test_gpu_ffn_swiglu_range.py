"""swiglu_quantize over the whole range of gates, the lowest and infinite ones among them: what it computes before it rounds is read from the scales of blocks (or rows)
that hold one value."""
import pytest
import torch

import ffn_reference as R

pytestmark = pytest.mark.gpu
FORMS = [("block", torch.int8), ("token", torch.int8), ("block", R.F8)]

# Units of 2^-24 of the value.  Gates from -87 on, fp32: ex2.approx 4 (two units in the last place), ln 2 in fp32 4 (its rounding, 1.9e-9, times an exponent of at most 126), 1 - r and
# 1 + e 2, the reciprocal 2 (one unit in the last place), two products 2, the scale's division 1; bf16: 1.6 for the square left out, not 4.
# Below: expf twice 8, four products, the sum and the division 5, the scale's division 1.
UNITS = 15


def _rel(gates, ups, scales, dtype, x, N=None):
    """Relative error of silu(gate) * up for each pair, each in a block (scales="token": a row) whose other ups are zero."""
    import gemm_int8_b200 as g

    gates, ups = gates.to(x), ups.to(x)
    n = gates.numel()
    per_row = 1 if scales == "token" else 8
    rows, N = n // per_row, N or 128 * per_row
    gen = torch.Generator(device="cuda").manual_seed(n)
    gu = torch.zeros(rows, 2 * N, device="cuda", dtype=x)
    gu[:, :N] = torch.randn(rows, N, generator=gen, device="cuda").to(x)
    row = torch.arange(n, device="cuda") // per_row
    col = torch.arange(n, device="cuda") % per_row * 128 + (torch.arange(n, device="cuda") * 37) % 128
    if scales == "token":
        col = (torch.arange(n, device="cuda") * 101) % N
    gu[row, col], gu[row, N + col] = gates, ups
    s = g.swiglu_quantize(gu, scales=scales, dtype=dtype)[1].reshape(-1).double() * R.TOP[dtype]
    if scales == "block":
        s = s[: n]
    v = gates.double() * torch.sigmoid(gates.double()) * ups.double()
    return (s - v.abs()).abs() / v.abs()


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lo,hi,up", [(-80.0, -65.0, 1.0), (-87.0, -80.0, 1e3), (-90.0, -86.0, 1e30), (-170.0, -88.0, 3e38), (1e30, 2e38, 1e-3)])
def test_value_of_one(lo, hi, up, x, scales, dtype):
    gen = torch.Generator(device="cuda").manual_seed(17)
    n = 4096
    gates = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * (hi - lo) + lo
    ups = up * (0.5 + 0.5 * torch.rand(n, generator=gen, device="cuda", dtype=torch.float64))
    rel = _rel(gates.float(), ups.float(), scales, dtype, x)
    assert float(rel.max()) <= UNITS * 2.0 ** -24, (float(rel.max()) * 2 ** 24, float(gates[rel.argmax()]))


@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
def test_value_of_one_in_rows_beyond_the_registers(x):
    """Rows of more than 32768 features with a scale per token are read twice behind the first 32768."""
    gen = torch.Generator(device="cuda").manual_seed(18)
    for lo, hi, up in ((-90.0, -80.0, 1e30), (-170.0, -90.0, 3e38)):
        gates = torch.rand(64, generator=gen, device="cuda") * (hi - lo) + lo
        rel = _rel(gates, torch.full((64,), up, device="cuda"), "token", torch.int8, x, N=40016)
        assert float(rel.max()) <= UNITS * 2.0 ** -24


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
def test_rows_of_low_gates(x, scales, dtype):
    """Every value of a row below -64, and such rows beside ordinary ones and beside NaN: each q against 64 bits."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(2)
    for N in (128, 1040, 36000):
        gate = torch.randn(6, N, generator=gen, device="cuda") * 3
        up = torch.randn(6, N, generator=gen, device="cuda")
        gate[1] = -80 - 7 * torch.rand(N, generator=gen, device="cuda")
        gate[2], up[2] = -87 - 2 * torch.rand(N, generator=gen, device="cuda"), up[2] * 1e30
        gate[3], up[3] = -100 - 60 * torch.rand(N, generator=gen, device="cuda"), up[3] * 1e37
        gate[4, ::2] = -88.0
        gu = torch.cat([gate, up], 1).to(x)
        q, s = g.swiglu_quantize(gu, scales=scales, dtype=dtype)
        v, _ = R.swiglu(gu)
        R.check_quantised(q, s, v, v.abs() * UNITS * 2.0 ** -24 + 2.0 ** -140, dtype, scales == "block")
        # an element's value does not depend on what stands beside it in other blocks, low gates and NaN among them
        if scales == "block" and N > 1024:
            other = gu.clone()
            other[0, 128], other[0, 300], other[0, 700] = -88.0, float("nan"), float("-inf")
            q2, s2 = g.swiglu_quantize(other, scales=scales, dtype=dtype)
            same = [0, 3, 4] + list(range(6, s.shape[1]))
            assert torch.equal(s2[0, same], s[0, same]) and torch.isnan(s2[0, [2, 5]]).all()
            assert torch.equal(q2[0, :128].view(torch.uint8), q[0, :128].view(torch.uint8)) and torch.equal(q2[0, 384:640].view(torch.uint8), q[0, 384:640].view(torch.uint8))


@pytest.mark.parametrize("scales,dtype", FORMS)
def test_infinite_and_largest_gates(scales, dtype):
    """What the definition gives: +inf and the largest finite gates pass through, -inf is NaN, a finite low gate times an infinite up is infinite."""
    import gemm_int8_b200 as g

    for x in (torch.bfloat16, torch.float32):
        gu = torch.ones(6, 2 * 128, device="cuda", dtype=x)
        gu[0, 5], gu[1, 5], gu[2, 5] = float("inf"), torch.finfo(x).max, float("-inf")
        gu[3, 5], gu[3, 128 + 5] = -70.0, float("inf")
        gu[4, 5], gu[4, 128 + 5] = torch.finfo(x).max, 0.5
        q, s = g.swiglu_quantize(gu, scales=scales, dtype=dtype)
        s = s.reshape(6).double() * R.TOP[dtype]
        assert torch.isinf(s[0]) and torch.isnan(s[2]) and torch.isinf(s[3])
        top = float(torch.finfo(x).max)
        assert abs(float(s[1]) / top - 1) <= UNITS * 2.0 ** -24 and abs(float(s[4]) / (0.5 * top) - 1) <= UNITS * 2.0 ** -24
        assert float(s[5]) > 0.7


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N", [(3, 640), (2500, 256), (5, 40016), (1300, 2064)])
def test_low_gates_among_ordinary_ones(M, N, x, scales, dtype):
    """Gates below -87 here and there, whose ups make their values too small to count, ones among the others, or the largest, in more rows than a CTA has and beside NaN: each
    q and scale against 64 bits, and rows without them as they are by themselves."""
    import gemm_int8_b200 as g

    gen = torch.Generator(device="cuda").manual_seed(M + N)
    gate, up = torch.randn(M, N, generator=gen, device="cuda"), torch.randn(M, N, generator=gen, device="cuda")
    kind = torch.randint(0, 5, (M,), generator=gen, device="cuda")  # 0 none, 1 too small, 2 among the others, 3 the largest, 4 NaN too
    for c in (7, N // 2 + 3, N - 1):
        low = -87.5 - 12 * torch.rand(M, generator=gen, device="cuda")
        size = torch.tensor([0.0, 1e-4, 0.3, 20.0, 0.3], device="cuda")[kind].double()
        u = (size / (low.double() * torch.sigmoid(low.double())).abs()).clamp(max=3e38).float()
        some = (kind > 0) & (torch.rand(M, generator=gen, device="cuda") < 0.7)
        gate[some, c], up[some, c] = low[some], u[some]
    gu = torch.cat([gate, up], 1).to(x)
    gu[kind == 4, 50] = float("nan")
    q, s = g.swiglu_quantize(gu, scales=scales, dtype=dtype)
    assert torch.isnan(s.reshape(M, -1)[kind == 4][:, 0]).all()
    fine = kind != 4
    v, _ = R.swiglu(gu[fine])
    R.check_quantised(q[fine], s[fine], v, v.abs() * UNITS * 2.0 ** -24 + 2.0 ** -140, dtype, scales == "block")
    plain = kind == 0
    alone = g.swiglu_quantize(gu[plain], scales=scales, dtype=dtype)
    assert torch.equal(alone[0].view(torch.uint8), q[plain].view(torch.uint8)) and torch.equal(alone[1], s[plain])


@pytest.mark.parametrize("scales,dtype", FORMS)
@pytest.mark.parametrize("x", [torch.bfloat16, torch.float32])
def test_lowest_gates_hide_no_other(x, scales, dtype):
    """Gates of the type's lowest value, as a mask would leave, give zeros and do not keep a low gate beside them, of one with a large up, from counting."""
    import gemm_int8_b200 as g

    N = 256
    for lowest in (torch.finfo(x).min, -1e38, -1e9):
        gu = torch.ones(4, 2 * N, device="cuda", dtype=x)
        gu[:, :N] = 0.25
        gu[0, 8:16] = lowest
        gu[1, 8:12], gu[1, 12], gu[1, N + 12] = lowest, -88.0, 1e37
        gu[2, 12], gu[2, N + 12] = -88.0, 1e37
        gu[3, 8:N:2] = lowest
        q, s = g.swiglu_quantize(gu, scales=scales, dtype=dtype)
        v, _ = R.swiglu(gu)
        assert float(v[1].abs().max()) > 3
        R.check_quantised(q, s, v, v.abs() * UNITS * 2.0 ** -24, dtype, scales == "block")
        assert not q[0, 8:16].float().any()
