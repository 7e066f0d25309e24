"""The experts' products, bit for bit against integer sums and three fp32 roundings; SwiGLU against 64 bits."""
import pytest
import torch

import experts_reference as R

pytestmark = pytest.mark.gpu


def _problem(counts, N, K, seed, gather=None, tail=0):
    """counts: rows per expert; gather: (tokens, top_k) or None; tail: rows that belong to nobody."""
    gen = torch.Generator().manual_seed(seed)
    E, kept = len(counts), sum(counts)
    offsets = torch.tensor([0] + list(counts), dtype=torch.int32).cumsum(0).int()
    slots = None
    rows_x = kept + tail
    k = 1
    if gather:
        rows_x, k = gather
        slots = torch.cat([torch.randint(0, rows_x * k, (kept,), generator=gen), torch.full((tail,), -1)]).int()
    x_q = torch.randint(-128, 128, (rows_x, K), dtype=torch.int8, generator=gen)
    w_q = torch.randint(-128, 128, (E, N, K), dtype=torch.int8, generator=gen)
    x_scale = torch.rand(rows_x, generator=gen) * 0.02 + 0.001
    w_scale = (torch.rand(E, N, generator=gen) * 0.9 + 0.1) / (127 * K ** 0.5)
    return x_q, w_q, x_scale, w_scale, offsets, slots, k


def _cuda(*ts):
    return [t.cuda() if isinstance(t, torch.Tensor) else t for t in ts]


def _check_product(problem):
    import gemm_int8_b200 as g

    out = g.matmul_experts(*_cuda(*problem))
    _, single = R.product(*problem)
    assert torch.equal(out.cpu(), single.to(torch.bfloat16))
    assert g.device_status() == 0


def _check_swiglu(problem):
    import gemm_int8_b200 as g

    out = g.matmul_experts_swiglu(*_cuda(*problem)).cpu().double()
    exact, _ = R.product(*problem)
    gate, h = R.swiglu(exact)
    # in units of 2^-24: three roundings each of gate and up (the gate's once more per unit of the exponent's argument), 4 + 2.35 |gate| (2 + 1.173
    # |gate| ulp) for the fast exponential, 1 for the sum, 2 (1 ulp) for the reciprocal, 3 for the products; one rounding to bf16; results below
    # what fp32 holds
    rel = 2 ** -8 * (1 + 2 ** -8) + (5.4 * gate.abs() + 16) * 2 ** -24
    assert ((out - h).abs() <= rel * h.abs() + 1e-36).all()
    assert g.device_status() == 0


# widths of the token tile: up to 32, 64, 128, 256 rows per expert, and more than one tile
COUNTS = [[1], [0, 1, 0], [3, 0, 17, 16, 1], [33, 0, 64, 1, 15], [100, 128, 0, 65], [129, 300, 0, 256, 257], [700, 5], [0, 0, 0]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("N,K", [(128, 128), (200, 400), (1, 16), (257, 1040)])
def test_contiguous_rows(counts, N, K):
    _check_product(_problem(counts, N, K, seed=N + len(counts)))
    _check_product(_problem(counts, N, K, seed=N, tail=19))


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("N,K", [(128, 256), (130, 144)])
@pytest.mark.parametrize("tokens,k", [(1, 1), (7, 3), (400, 8)])
def test_gathered_rows(counts, N, K, tokens, k):
    _check_product(_problem(counts, N, K, seed=tokens, gather=(tokens, k)))
    _check_product(_problem(counts, N, K, seed=tokens, gather=(tokens, k), tail=5))


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("inner,K", [(64, 128), (100, 272), (1, 16), (129, 1040)])
def test_swiglu(counts, inner, K):
    _check_swiglu(_problem(counts, 2 * inner, K, seed=inner))
    _check_swiglu(_problem(counts, 2 * inner, K, seed=inner, gather=(50, 2), tail=9))


def test_large_groups_over_many_tiles():
    """More tiles than CTAs, several accumulator rounds per CTA, all tile widths."""
    gen = torch.Generator().manual_seed(4)
    for rows in (6, 40, 100, 300):
        counts = torch.randint(0, 2 * rows, (24,), generator=gen).tolist()
        _check_product(_problem(counts, 1400, 384, seed=rows, gather=(3 * rows, 4)))
        _check_swiglu(_problem(counts, 1400, 384, seed=rows))


@pytest.mark.parametrize("counts", [[1, 1], [0, 3, 0, 17, 1], [32], [40, 1]], ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("K", [6144, 6160])
def test_few_long_tiles(counts, K):
    """Fewer weight tiles than SMs and a long K: the form with a deep ring (and, with more rows, the ordinary one)."""
    _check_product(_problem(counts, 200, K, seed=K))
    _check_product(_problem(counts, 200, K, seed=K, gather=(3, 2), tail=2))
    _check_swiglu(_problem(counts, 160, K, seed=K))
    _check_swiglu(_problem(counts, 160, K, seed=K, gather=(3, 2), tail=2))


def test_rows_of_nobody_are_zero():
    """Rows in front of the first expert's and behind the last one's, over memory that held something else."""
    import gemm_int8_b200 as g

    for N in (128, 130):
        x_q, w_q, x_scale, w_scale, offsets, _, _ = _problem([5, 40], N, 64, seed=N, tail=30)
        offsets = offsets + 11
        junk = torch.full((75, N), 9.0, dtype=torch.bfloat16, device="cuda")  # (the allocator hands this memory to the result)
        del junk
        out = g.matmul_experts(*_cuda(x_q, w_q, x_scale, w_scale, offsets)).cpu()
        _, single = R.product(x_q, w_q, x_scale, w_scale, offsets)
        assert torch.equal(out, single.to(torch.bfloat16)) and (out[:11] == 0).all() and (out[56:] == 0).all() and (out[11:56] != 0).any()


def test_extreme_operands():
    """The largest sums there are, scales of zero, infinity and NaN in a row of their own."""
    import gemm_int8_b200 as g

    K = 4096
    x_q = torch.full((40, K), -128, dtype=torch.int8)
    w_q = torch.full((2, 128, K), -128, dtype=torch.int8)
    w_q[1] = 127
    x_scale = torch.ones(40)
    x_scale[3], x_scale[4], x_scale[5] = 0.0, float("inf"), float("nan")
    w_scale = torch.full((2, 128), 0.5)
    offsets = torch.tensor([0, 20, 40], dtype=torch.int32)
    out = g.matmul_experts(*_cuda(x_q, w_q, x_scale, w_scale, offsets)).cpu()
    _, single = R.product(x_q, w_q, x_scale, w_scale, offsets)
    assert torch.equal(out.nan_to_num(7.0), single.to(torch.bfloat16).nan_to_num(7.0))


def test_silu_far_out():
    """Gates of up to a thousand in magnitude."""
    K = 128
    x_q = torch.full((8, K), 127, dtype=torch.int8)
    w_q = torch.randint(-127, 128, (1, 128, K), dtype=torch.int8, generator=torch.Generator().manual_seed(0))
    w_q[0, :64] = (torch.arange(64) * 4 - 127)[:, None].to(torch.int8)
    x_scale = torch.logspace(-6, -3.3, 8)
    problem = (x_q, w_q, x_scale, torch.ones(1, 128), torch.tensor([0, 8], dtype=torch.int32), None, 1)
    _check_swiglu(problem)


def test_offsets_and_slots_out_of_range_stay_in_bounds():
    """Wrong offsets or slots give wrong rows and nothing else (they are clamped before anything is addressed)."""
    import gemm_int8_b200 as g

    x_q, w_q, x_scale, w_scale, offsets, slots, k = _cuda(*_problem([20, 30, 14], 128, 128, seed=1, gather=(40, 2)))
    for bad in ([0, 50, 20, 64], [-5, 10, 2 ** 31 - 1, 64], [64, 0, 64, 0], [0, 0, 0, 1000]):
        g.matmul_experts(x_q, w_q, x_scale, w_scale, torch.tensor(bad, dtype=torch.int32, device="cuda"), slots, k)
    g.matmul_experts(x_q, w_q, x_scale, w_scale, offsets, slots + 2 ** 30, k)
    g.matmul_experts(x_q, w_q, x_scale, w_scale, offsets, -slots, k)
    assert g.device_status() == 0
