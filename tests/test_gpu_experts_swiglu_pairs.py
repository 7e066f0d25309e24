"""SwiGLU with gathered rows on tiles of CTA pairs, the first product of a layer of prompts: against 64 bits."""
import pytest
import torch

from test_gpu_experts_product import _check_swiglu, _problem

pytestmark = pytest.mark.gpu

# (more than 64 rows per expert on average, out of more than 64 tokens: the two-CTA form)
COUNTS = [[100, 128, 0, 65], [129, 300, 0, 256, 257], [700, 5], [513], [33, 400, 31, 1, 64, 500]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("inner,K", [(64, 128), (100, 272), (128, 1040), (129, 1040), (257, 784), (1, 16)])
@pytest.mark.parametrize("tail", [0, 9])
def test_gathered(counts, inner, K, tail):
    """inner a multiple of 16 and not; K beyond the six stages of the ring."""
    _check_swiglu(_problem(counts, 2 * inner, K, seed=inner, gather=(400, 8), tail=tail))


@pytest.mark.parametrize("rows", [100, 300])
def test_gathered_over_many_tiles(rows):
    counts = torch.randint(0, 2 * rows, (24,), generator=torch.Generator().manual_seed(rows)).tolist()
    _check_swiglu(_problem(counts, 1400, 1040, seed=rows, gather=(3 * rows, 4)))
    _check_swiglu(_problem(counts, 1376, 400, seed=rows + 1, gather=(3 * rows, 4), tail=40))
