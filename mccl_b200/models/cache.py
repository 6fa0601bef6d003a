"""Keys and values of many sequences in pages of one allocation.

A page holds ``page_size`` neighbouring positions of one sequence in every layer, so that one page number stands for its keys and values
everywhere: ``pages`` is ``[layers, 2, pages, kv_heads, page_size, head_dim]``.  Which pages a sequence has is kept on the host (lists and counts of
owners) and, for the kernels, in ``table`` (int32 ``[sequences, width]``, -1 where there is none) and ``lengths`` (int32) on the device.  Changes of the
table are ordered on the current stream, like everything that reads it.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch

from .. import ops


class PagedKVCache:
    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, pages: int, max_sequences: int, max_positions: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, value in (("layers", layers), ("kv_heads", kv_heads), ("pages", pages), ("max_sequences", max_sequences), ("max_positions", max_positions),
                            ("page_size", page_size)):
            if value < 1:
                raise RuntimeError(f"PagedKVCache: {name} must be positive, got {value}")
        if head_dim < 1 or head_dim % 8:
            raise RuntimeError(f"PagedKVCache: head_dim must be a positive multiple of 8, got {head_dim}")
        self.page_size, self.max_positions, self.max_sequences = page_size, max_positions, max_sequences
        self.pages = torch.empty(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        width = -(-max_positions // page_size)
        self.table = torch.full((max_sequences, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_sequences, dtype=torch.int32, device=device)
        self._owners = [0] * pages                       # sequences that have the page
        self._free = list(range(pages - 1, -1, -1))      # the lowest page is taken first
        self._rows: Dict[int, List[int]] = {}            # row -> its pages in order, -1 where one was dropped
        self._length: Dict[int, int] = {}
        self._window: Dict[int, int] = {}                # row -> the window that pages were dropped for
        self._dropped: Dict[int, tuple] = {}             # row -> (i, j): nothing is left to drop among its pages i to j - 1

    # ------------------------------------------------------------------------------------------------------- what there is --
    @property
    def device(self) -> torch.device:
        return self.pages.device

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def rows(self) -> List[int]:
        return sorted(self._rows)

    def length(self, row: int) -> int:
        self._known(row)
        return self._length[row]

    def row_pages(self, row: int) -> List[int]:
        """The pages of a sequence in order (-1: dropped)."""
        self._known(row)
        return list(self._rows[row])

    def keys(self, layer: int) -> torch.Tensor:
        return self.pages[layer, 0]

    def values(self, layer: int) -> torch.Tensor:
        return self.pages[layer, 1]

    def _known(self, row: int) -> None:
        if row not in self._rows:
            raise RuntimeError(f"PagedKVCache: there is no sequence in row {row}")

    # ------------------------------------------------------------------------------------------------------------- changes --
    def add(self) -> int:
        """A new, empty sequence; returns its row."""
        return self._add_rows(1)[0]

    def _add_rows(self, n: int) -> List[int]:
        new = [r for r in range(self.max_sequences) if r not in self._rows][:n]
        if len(new) < n:
            raise RuntimeError(f"PagedKVCache: all {self.max_sequences} rows are taken")
        for r in new:
            self._rows[r], self._length[r] = [], 0
        return new

    def reserve(self, rows: Sequence[int], lengths: Sequence[int]) -> None:
        """Pages for the first ``lengths[i]`` positions of each sequence.  Nothing changes when there are not enough."""
        need: Dict[int, int] = {}
        for row, length in zip(rows, lengths):
            self._known(row)
            if length > self.max_positions:
                raise RuntimeError(f"PagedKVCache: {length} positions, at most {self.max_positions} were asked for")
            need[row] = max(need.get(row, 0), -(-length // self.page_size) - len(self._rows[row]))   # a row may be named more than once
        if sum(need.values()) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(need.values())} pages needed, {len(self._free)} of {len(self._owners)} free")
        at, new = [], []
        for row, n in need.items():
            for _ in range(n):
                page = self._free.pop()
                self._owners[page] = 1
                at.append((row, len(self._rows[row])))
                new.append(page)
                self._rows[row].append(page)
        self._write(at, new)

    def advance(self, rows: Sequence[int], count: int) -> None:
        """Notes on the host that each sequence has `count` more positions (``lengths`` is the caller's: kernels that append know it first)."""
        if count < 0:
            raise RuntimeError(f"PagedKVCache: {count} more positions; set_length() makes a sequence shorter")
        for row in rows:
            self._known(row)
            if -(-(self._length[row] + count) // self.page_size) > len(self._rows[row]):
                raise RuntimeError(f"PagedKVCache: row {row} has no pages for {self._length[row] + count} positions")
        for row in rows:
            self._length[row] += count

    def set_length(self, row: int, length: int) -> None:
        """The sequence's length, on the host and on the device.  A sequence that goes back among pages it shares keeps the whole ones before its new
        end; of the one that holds the end it gets a copy, and those behind it are the others' from then on (``reserve`` gives new ones).  It cannot
        go back to where ``drop_unseen`` has given back some of its window's last positions."""
        self._known(row)
        if length < 0 or -(-length // self.page_size) > len(self._rows[row]):
            raise RuntimeError(f"PagedKVCache: row {row} has no pages for {length} positions")
        if length < self._length[row]:
            self._go_back(row, length)
        self._length[row] = length
        self.lengths[row] = length

    def fork(self, row: int, count: int = 1) -> List[int]:
        """`count` new sequences that begin as this one.  Full pages are shared; the last one, which will be written, is copied."""
        self._known(row)
        if count < 0:
            raise RuntimeError(f"PagedKVCache: {count} forks")
        length, old = self._length[row], self._rows[row]
        full = length // self.page_size
        partial = old[full] if length % self.page_size else None
        if partial is not None and count > len(self._free):
            raise RuntimeError(f"PagedKVCache: {count} pages needed, {len(self._free)} of {len(self._owners)} free")
        new = self._add_rows(count)
        copies = []
        for r in new:
            pages = old[:full]
            for page in pages:
                if page >= 0:
                    self._owners[page] += 1
            if partial is not None:
                page = self._free.pop()
                self._owners[page] = 1
                copies.append(page)
                pages = pages + [page]
            self._rows[r], self._length[r] = pages, length
            if row in self._window:
                self._window[r] = self._window[row]
            if row in self._dropped:
                self._dropped[r] = self._dropped[row]
        self._write([(r, i) for r in new for i in range(len(self._rows[r]))], [page for r in new for page in self._rows[r]])
        self.lengths[self._indices(new)] = length
        if copies:
            ops.copy_pages(self.pages, self._numbers([partial] * len(copies)), self._numbers(copies), dim=2)
        return new

    def free(self, row: int) -> None:
        """The sequence goes, and with it the pages that it alone has."""
        self._known(row)
        for page in self._rows[row]:
            self._drop(page)
        del self._rows[row], self._length[row]
        self._window.pop(row, None)
        self._dropped.pop(row, None)
        self.table[row] = -1
        self.lengths[row] = 0

    def drop_unseen(self, rows: Sequence[int], window: int, sinks: int = 0) -> int:
        """Gives back pages none of whose positions a window of the last `window` positions and the first `sinks` sees, now or later; returns how many."""
        if window < 1 or sinks < 0:
            raise RuntimeError(f"PagedKVCache: no window of {window} with {sinks} first positions")
        at, dropped = [], 0
        for row in rows:
            self._known(row)
            first = self._length[row] - window   # the next token's window begins one later
            start, stop = -(-sinks // self.page_size), max(0, first) // self.page_size
            done, until = self._dropped.get(row, (start, start))   # what the steps before have walked over
            if done <= start <= until:
                look, self._dropped[row] = range(until, stop), (done, max(until, stop))
            else:
                look, self._dropped[row] = range(start, stop), (start, max(start, stop))
            for i in look:
                page = self._rows[row][i]
                if page >= 0:
                    dropped += self._drop(page)
                    self._rows[row][i] = -1
                    self._window[row] = window
                    at.append((row, i))
        self._write(at, [-1] * len(at))
        return dropped

    def compact(self) -> int:
        """Moves pages so that those in use are the first ones; returns how many there are.  One kernel moves all layers' keys and values."""
        used = sum(1 for n in self._owners if n)
        high = [page for page in range(used, len(self._owners)) if self._owners[page]]
        low = [page for page in range(used) if not self._owners[page]]
        moves = dict(zip(high, low))   # sources and places do not overlap
        if moves:
            ops.copy_pages(self.pages, self._numbers(high), self._numbers(low), dim=2)
            at, new = [], []
            for row, pages in self._rows.items():
                for i, page in enumerate(pages):
                    if page in moves:
                        pages[i] = moves[page]
                        at.append((row, i))
                        new.append(pages[i])
            self._write(at, new)
            for source, place in moves.items():
                self._owners[place], self._owners[source] = self._owners[source], 0
        self._free = list(range(len(self._owners) - 1, used - 1, -1))
        return used

    # -------------------------------------------------------------------------------------------------------------- inside --
    def _go_back(self, row: int, length: int) -> None:
        """No page that the sequence will write from position `length` on has another owner or was dropped.  (``fork`` shares pages in front of both
        sequences' ends only, and those that are dropped lie there too, so this is where such a page can come to lie behind one.)"""
        pages = self._rows[row]
        if row in self._window and any(page < 0 for page in pages[max(0, length - self._window[row]) // self.page_size:-(-length // self.page_size)]):
            raise RuntimeError(f"PagedKVCache: row {row} cannot go back to {length} positions, pages of its last {self._window[row]} were given back")
        full, end = length // self.page_size, -(-length // self.page_size)
        if row in self._dropped:
            self._dropped[row] = tuple(min(i, full) for i in self._dropped[row])
        own = [page for page in pages[end:] if page >= 0 and self._owners[page] == 1]
        cut = pages[full] if end > full and pages[full] >= 0 and self._owners[pages[full]] > 1 else None
        if cut is None and len(own) == len(pages) - end:
            return
        if cut is not None:
            if not own and not self._free:
                raise RuntimeError(f"PagedKVCache: 1 page needed, 0 of {len(self._owners)} free")
            copy = own.pop(0) if own else self._free.pop()
            ops.copy_pages(self.pages, self._numbers([cut]), self._numbers([copy]), dim=2)
        kept = pages[:full] + ([] if end == full else [pages[full] if cut is None else copy]) + own
        for page in pages[full:]:
            if page >= 0 and self._owners[page] > 1:
                self._owners[page] -= 1
        if cut is not None:
            self._owners[copy] = 1
        self._rows[row] = kept
        self._write([(row, i) for i in range(full, len(pages))], kept[full:] + [-1] * (len(pages) - len(kept)))

    def _drop(self, page: int) -> int:
        if page < 0:
            return 0
        self._owners[page] -= 1
        if self._owners[page] == 0:
            self._free.append(page)
            return 1
        return 0

    def _numbers(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.device)

    def _indices(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int64).to(self.device)

    def _write(self, at, pages: Optional[Sequence[int]]) -> None:
        """table[row, i] = page for all (row, i)."""
        if at:
            flat = self._indices([row * self.table.shape[1] + i for row, i in at])
            self.table.view(-1)[flat] = self._numbers(pages)
