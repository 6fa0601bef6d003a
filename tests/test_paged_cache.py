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


def test_a_shortened_fork_leaves_the_others_alone():
    for back in (6, 4, 3, 1, 0):
        cache = cache_of(pages=12)
        a = cache.add()
        kv = fill(cache, a, 8, 1)
        b, c = cache.fork(a, 2)
        cache.set_length(b, back)
        sound(cache)
        assert torch.equal(read(cache, b), kv[:, :, :back]) if back else True
        cache.reserve([b], [11])
        for i in range(back, 11):
            append(cache, b, i, float(i))
        cache.set_length(b, 11)
        sound(cache)
        assert torch.equal(read(cache, a), kv) and torch.equal(read(cache, c), kv)
        assert torch.equal(read(cache, b)[:, :, :back], kv[:, :, :back])
        assert all((read(cache, b)[:, :, i] == i).all() for i in range(back, 11))
        assert len(set(cache.row_pages(b)) & set(cache.row_pages(a))) == back // 4


def test_the_first_one_of_a_fork_may_go_back_too():
    cache = cache_of(pages=12)
    a = cache.add()
    kv = fill(cache, a, 10, 2)
    (b,) = cache.fork(a)
    cache.reserve([a], [16])
    cache.set_length(a, 2)      # a page that is shared in part, one that is shared behind, and two of its own
    sound(cache)
    cache.reserve([a], [16])
    for i in range(2, 16):
        append(cache, a, i, 1.0)
    cache.set_length(a, 16)
    sound(cache)
    assert torch.equal(read(cache, b), kv) and torch.equal(read(cache, a)[:, :, :2], kv[:, :, :2]) and (read(cache, a)[:, :, 2:] == 1).all()


def test_pages_of_its_own_stay_where_a_sequence_goes_back():
    cache = cache_of(pages=4)
    a = cache.add()
    kv = fill(cache, a, 16, 3)
    pages = cache.row_pages(a)
    cache.set_length(a, 5)
    assert cache.row_pages(a) == pages and cache.free_pages == 0 and torch.equal(read(cache, a), kv[:, :, :5])
    sound(cache)


def test_going_back_without_a_page_to_copy_to_changes_nothing():
    cache = cache_of(pages=2)
    a = cache.add()
    kv = fill(cache, a, 8, 4)
    (b,) = cache.fork(a)
    with pytest.raises(RuntimeError, match="PagedKVCache"):
        cache.set_length(b, 6)
    sound(cache)
    assert cache.length(b) == 8 and torch.equal(read(cache, a), kv) and torch.equal(read(cache, b), kv)
    cache.set_length(b, 4)      # whole pages need no copy
    sound(cache)
    cache.free(a)
    assert torch.equal(read(cache, b), kv[:, :, :4])


def test_the_host_count_goes_forward_only():
    cache = cache_of()
    a = cache.add()
    fill(cache, a, 8, 5)
    with pytest.raises(RuntimeError, match="set_length"):
        cache.advance([a], -2)
    assert cache.length(a) == 8


def windowed():
    """27 positions in pages of 4, of which a window of 10 and one first position have left the pages 0 and 4 to 6."""
    cache = cache_of(pages=12, rows=2)
    a = cache.add()
    kv = fill(cache, a, 27, 6)
    assert cache.drop_unseen([a], 10, 1) == 3 and cache.row_pages(a)[1:4] == [-1] * 3
    return cache, a, kv


@pytest.mark.parametrize("length", [25, 24, 17, 16, 15, 9, 6, 5])
def test_no_way_back_to_where_a_window_is_gone(length):
    cache, a, _ = windowed()
    before = cache.row_pages(a)
    with pytest.raises(RuntimeError, match="given back"):
        cache.set_length(a, length)
    assert cache.length(a) == 27 and cache.row_pages(a) == before
    sound(cache)


@pytest.mark.parametrize("length", [26, 4, 2, 0])
def test_back_to_where_everything_is_there(length):
    cache, a, kv = windowed()
    cache.set_length(a, length)
    sound(cache)
    end = min(length + 13, 32)
    cache.reserve([a], [end])
    for i in range(length, end):
        append(cache, a, i, float(i))
    cache.set_length(a, end)
    sound(cache)
    for i in list(range(min(length, 4))) + list(range(16 if length > 4 else length, end)):
        page = int(cache.table[a, i // 4])
        assert page >= 0
        held = cache.pages[:, :, page, :, i % 4]
        assert torch.equal(held, kv[:, :, i]) if i < length else (held == i).all()
    (b,) = cache.fork(a)
    sound(cache)


def test_a_fork_knows_what_its_window_is():
    cache, a, _ = windowed()
    (b,) = cache.fork(a)
    with pytest.raises(RuntimeError, match="given back"):
        cache.set_length(b, 20)
    cache.set_length(b, 3)
    sound(cache)


def test_counts_and_windows_that_make_no_sense():
    cache = cache_of(rows=4)
    a = cache.add()
    kv = fill(cache, a, 16, 7)
    for call in (lambda: cache.fork(a, -1), lambda: cache.drop_unseen([a], 0), lambda: cache.drop_unseen([a], -4), lambda: cache.drop_unseen([a], 2, -5)):
        with pytest.raises(RuntimeError, match="PagedKVCache"):
            call()
        sound(cache)
        assert cache.rows == [a] and torch.equal(read(cache, a), kv)
    assert cache.fork(a, 0) == []


class Counted(list):
    looks = 0

    def __getitem__(self, i):
        Counted.looks += 1
        return super().__getitem__(i)


def test_pages_out_of_sight_are_looked_at_once():
    cache = PagedKVCache(1, 1, 8, pages=600, max_sequences=2, max_positions=2400, page_size=4, device="cpu")
    a = cache.add()
    cache.reserve([a], [2000])
    cache.set_length(a, 2000)
    cache._rows[a] = Counted(cache._rows[a])
    assert cache.drop_unseen([a], 100, 5) == 475 - 2      # positions below 1900, without the first two pages
    Counted.looks = 0
    for n in range(2001, 2101):
        cache.reserve([a], [n])
        cache.set_length(a, n)
        cache.drop_unseen([a], 100, 5)
    assert cache.row_pages(a).count(-1) == 500 - 2 and Counted.looks <= 3 * 100
    sound(cache)


def test_what_is_out_of_sight_is_given_back_whatever_was_asked_before():
    """A walk that begins where the last one ended gives back what a walk over everything does."""
    def unseen(pages, length, window, sinks):
        return [p for i, p in enumerate(pages) if p >= 0 and -(-sinks // 4) <= i < max(0, length - window) // 4]

    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        cache = PagedKVCache(1, 1, 8, pages=200, max_sequences=3, max_positions=200, page_size=4, device="cpu")
        rows = [cache.add()]
        for _ in range(60):
            row = rows[int(torch.randint(0, len(rows), (1,), generator=g))]
            kind = int(torch.randint(0, 8, (1,), generator=g))
            length = cache.length(row)
            if kind == 0 and len(rows) < 3:
                rows += cache.fork(row)
            elif kind == 1 and length:
                to = int(torch.randint(0, length, (1,), generator=g))
                try:
                    cache.set_length(row, to)
                except RuntimeError:
                    pass
            elif kind <= 4 and length < 190:
                to = length + int(torch.randint(1, 10, (1,), generator=g))
                cache.reserve([row], [to])
                cache.set_length(row, to)
            else:
                window, sinks = int(torch.randint(1, 40, (1,), generator=g)), int(torch.randint(0, 30, (1,), generator=g)) * int(torch.randint(0, 2, (1,), generator=g))
                want = unseen(cache.row_pages(row), cache.length(row), window, sinks)
                free = cache.free_pages
                got = cache.drop_unseen([row], window, sinks)
                assert not unseen(cache.row_pages(row), cache.length(row), window, sinks)
                assert got == cache.free_pages - free <= len(want)
            sound(cache)
