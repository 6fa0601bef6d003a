"""The paged cache's bookkeeping where sequences share pages, go back, or are named more than once."""
import pytest
import torch

from mccl_b200 import ops
from mccl_b200.models import PagedKVCache
from tests.test_generate import cache_of, fill, read


def append(cache, row, at, value):
    """A token with this value at position `at` of a sequence, in all layers."""
    one = torch.full((1, 2, 8), value).half()
    for i in range(cache.pages.shape[0]):
        ops.paged_append(one, one, cache.keys(i), cache.values(i), cache.table, torch.tensor([at], dtype=torch.int32), rows=torch.tensor([row], dtype=torch.int32))


def sound(cache):
    """The table is what the host has, every page has as many owners as sequences that list it, and the others are free."""
    count = [0] * cache.pages.shape[2]
    for row in range(cache.max_sequences):
        pages = cache.row_pages(row) if row in cache.rows else []
        assert cache.table[row].tolist() == pages + [-1] * (cache.table.shape[1] - len(pages))
        assert cache.lengths[row] == (cache.length(row) if row in cache.rows else 0)
        for page in pages:
            if page >= 0:
                count[page] += 1
    assert count == cache._owners and sorted(cache._free) == [p for p, n in enumerate(count) if n == 0]


def test_a_row_that_is_named_twice_gets_its_pages_once():
    for row in (0, 2):
        cache = PagedKVCache(1, 1, 8, pages=10, max_sequences=3, max_positions=8, page_size=4, device="cpu")
        rows = [cache.add() for _ in range(3)]
        cache.reserve(rows, [4, 4, 4])
        cache.reserve([row, row, row], [8, 5, 8])
        sound(cache)
        assert len(cache.row_pages(row)) == 2 and cache.free_pages == 6
