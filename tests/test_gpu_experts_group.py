"""Grouping by expert: a stable counting sort, equal to the plain one in every element."""
import pytest
import torch

import experts_reference as R

pytestmark = pytest.mark.gpu


def _check(experts, E, first=0):
    import gemm_int8_b200 as g

    got = g.group_by_expert(experts.cuda(), E, first)
    flat = experts.reshape(-1).long() - first
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(key, minlength=E + 1)[:E].cumsum(0)]).int()
    order = torch.argsort(key, stable=True).int()
    slots = torch.where(torch.arange(flat.numel()) < offsets[E], order, -1)
    places = torch.full((flat.numel(),), -1, dtype=torch.int32)
    kept = int(offsets[E])
    places[order[:kept].long()] = torch.arange(kept, dtype=torch.int32)
    for a, b in zip(got, (offsets, slots.int(), places.reshape(experts.shape))):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)
    return got


@pytest.mark.parametrize("T,k", [(0, 2), (1, 1), (1, 8), (5, 3), (61, 4), (255, 8), (256, 8), (257, 8), (700, 6), (1500, 5), (4097, 8)])
@pytest.mark.parametrize("E", [1, 7, 64, 256, 1024])
def test_sizes(T, k, E):
    experts = torch.randint(0, E, (T, k), dtype=torch.int32, generator=torch.Generator().manual_seed(T + E))
    got = _check(experts, E)
    if T <= 61 and E <= 64:
        for a, b in zip(got, R.group(experts, E)):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("T", [3, 300, 9000])
def test_ids_of_nobody_and_of_other_ranks(T):
    gen = torch.Generator().manual_seed(T)
    experts = torch.randint(-1, 40, (T, 4), dtype=torch.int32, generator=gen)
    experts[0, 0] = 2 ** 31 - 1
    experts[-1, -1] = -2 ** 31
    for E, first in ((40, 0), (10, 0), (10, 30), (7, 13), (5, 100)):
        _check(experts, E, first)


@pytest.mark.parametrize("T", [40, 9000])
def test_one_expert_takes_all_and_none_takes_any(T):
    _check(torch.full((T, 2), 3, dtype=torch.int32), 8)
    _check(torch.full((T, 2), -1, dtype=torch.int32), 8)


def test_large_and_strided():
    gen = torch.Generator().manual_seed(9)
    _check(torch.randint(0, 512, (70001, 9), dtype=torch.int32, generator=gen), 512)
    _check(torch.randint(-1, 1024, (20001, 8), dtype=torch.int32, generator=gen), 1024)
    _check(torch.randint(0, 3, (30000, 8), dtype=torch.int32, generator=gen), 3)
    _check(torch.randint(0, 16, (300, 16), dtype=torch.int32, generator=gen)[:, 3:9], 16)
