"""PagedCache.slots at the edges of a page table, on the CPU."""
import pytest
import torch

import bitween_amd as bw


@pytest.fixture
def cache():
    return bw.PagedCache(3, 2, 64, 16, device="cpu")


@pytest.mark.parametrize("positions", [[0, 5], [-1, 100]])
def test_a_table_without_pages_has_padding_only(cache, positions):
    table = torch.empty(2, 0, dtype=torch.int32)
    positions = torch.tensor(positions)
    got = cache.slots(table, positions)
    assert got.dtype == torch.int64 and got.tolist() == [-1, -1]
    got = cache.slots(table, positions.int(), torch.tensor([1, 1]))
    assert got.dtype == torch.int64 and got.tolist() == [-1, -1]


def test_no_tokens_and_no_sequences(cache):
    none = torch.empty(0, dtype=torch.int64)
    assert cache.slots(torch.empty(0, 4, dtype=torch.int32), none).tolist() == []
    assert cache.slots(torch.empty(2, 0, dtype=torch.int32), none, none).tolist() == []
    assert cache.slots(torch.zeros(2, 4, dtype=torch.int32), none, none).dtype == torch.int64
