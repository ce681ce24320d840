"""Host-side accounting of a paged cache: which pages hold which tokens.

No device work happens here; ``PagedKVCache`` turns the page copies that the
methods return into launches.
"""

from __future__ import annotations

from typing import Sequence

import numpy as np

__all__ = ["PageTable"]


class PageTable:
    """Pages of up to ``max_sequences`` sequences over a pool of ``n_pages``.

    Full pages may be shared by forked sequences (reference counts); a page
    that takes new tokens belongs to one sequence, so ``extend`` gives a
    sequence its own copy of a shared last page first (the ``(src, dst)`` pairs
    it returns).  ``table[row, i]`` is the page of tokens ``[i * page_size, (i +
    1) * page_size)``; ``dirty`` collects the entries that changed.  Every
    method checks its arguments before it changes anything.
    """

    def __init__(self, n_pages: int, page_size: int, max_sequences: int, max_tokens: int) -> None:
        self.n_pages, self.page_size, self.max_sequences = int(n_pages), int(page_size), int(max_sequences)
        if self.n_pages < 1 or self.max_sequences < 1 or int(max_tokens) < 1:
            raise ValueError("PageTable: n_pages, max_sequences and max_tokens must be positive")
        if self.n_pages > 2 ** 31 - 1 or int(max_tokens) > 2 ** 31 - 257:
            raise ValueError("PageTable: pages and tokens are counted in 32 bits")
        self.max_pages = -(-int(max_tokens) // self.page_size)
        self.max_tokens = int(max_tokens)
        self.table = np.zeros((self.max_sequences, self.max_pages), dtype=np.int32)
        self.dirty: list[tuple[int, int, int]] = []  # (row, first, last + 1)
        self.refs = np.zeros(self.n_pages, dtype=np.int32)
        self._free = list(range(self.n_pages - 1, -1, -1))
        self._rows = list(range(self.max_sequences - 1, -1, -1))
        self._seqs: dict[int, list[int]] = {}  # id -> [row, length, pages]
        self._next = 0
        self.epoch = 0  # grows when pages or lengths of existing sequences change hands

    # ---- queries ---------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def sequences(self) -> list[int]:
        return list(self._seqs)

    def _get(self, seq: int) -> list[int]:
        try:
            return self._seqs[seq]
        except (KeyError, TypeError):
            raise KeyError(f"sequence {seq!r} is not in the cache") from None

    def row(self, seq: int) -> int:
        return self._get(seq)[0]

    def length(self, seq: int) -> int:
        return self._get(seq)[1]

    def pages(self, seq: int) -> list[int]:
        row, _, n = self._get(seq)
        return self.table[row, :n].tolist()

    # ---- changes ---------------------------------------------------------

    def add(self) -> int:
        """A new empty sequence."""
        if not self._rows:
            raise RuntimeError(f"all {self.max_sequences} sequences are in use")
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = [self._rows.pop(), 0, 0]
        return seq

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> list[tuple[int, int]]:
        """Room for ``counts[i]`` more tokens of ``seqs[i]``; the page copies to make first."""
        if len(seqs) != len(counts):
            raise ValueError(f"{len(seqs)} sequences but {len(counts)} token counts")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        size, need, shared = self.page_size, 0, {}
        plan = []
        for seq, n in zip(seqs, counts):
            ent = self._get(seq)
            row, length, pages = ent
            n = int(n)
            if n < 0:
                raise ValueError(f"token counts must not be negative (got {n})")
            if length + n > self.max_tokens:
                raise ValueError(f"sequence {seq}: {length} + {n} tokens exceed max_tokens = {self.max_tokens}")
            fresh = -(-(length + n) // size) - pages
            copy = -1
            if n > 0 and length % size:  # the last page takes tokens: it must be this sequence's own
                last = int(self.table[row, pages - 1])
                left = shared.get(last, int(self.refs[last]))
                if left > 1:
                    shared[last] = left - 1
                    copy = last
            need += fresh + (copy >= 0)
            plan.append((ent, n, fresh, copy))
        if need > len(self._free):
            raise RuntimeError(f"out of pages: {need} needed, {len(self._free)} free")
        copies = []
        for ent, n, fresh, copy in plan:
            row, length, pages = ent
            if copy >= 0:
                page = self._take()
                self.refs[copy] -= 1
                self.table[row, pages - 1] = page
                self.dirty.append((row, pages - 1, pages))
                copies.append((copy, page))
            if fresh > 0:
                got = self._free[-fresh:][::-1]
                del self._free[-fresh:]
                self.refs[got] = 1
                self.table[row, pages:pages + fresh] = got
                self.dirty.append((row, pages, pages + fresh))
                ent[2] = pages + fresh
            ent[1] = length + n
        return copies

    def _take(self) -> int:
        page = self._free.pop()
        self.refs[page] = 1
        return page

    def fork(self, seq: int) -> int:
        """A new sequence with ``seq``'s tokens, on the same pages."""
        row, length, pages = self._get(seq)
        new = self.add()
        ent = self._seqs[new]
        self.table[ent[0], :pages] = self.table[row, :pages]
        self.refs[self.table[row, :pages]] += 1
        if pages:
            self.dirty.append((ent[0], 0, pages))
        ent[1], ent[2] = length, pages
        self.epoch += 1
        return new

    def _release(self, row: int, first: int, last: int) -> None:
        for page in self.table[row, first:last].tolist()[::-1]:
            self.refs[page] -= 1
            if self.refs[page] == 0:
                self._free.append(page)

    def truncate(self, seq: int, length: int) -> None:
        """Drop ``seq``'s tokens from ``length`` on (rejected drafts)."""
        ent = self._get(seq)
        length = int(length)
        if not 0 <= length <= ent[1]:
            raise ValueError(f"sequence {seq} has {ent[1]} tokens: cannot keep {length}")
        keep = -(-length // self.page_size)
        self._release(ent[0], keep, ent[2])
        ent[1], ent[2] = length, keep
        self.epoch += 1

    def free(self, seq: int) -> None:
        """Forget ``seq`` and give back the pages no other sequence holds."""
        row, _, pages = self._get(seq)
        self._release(row, 0, pages)
        del self._seqs[seq]
        self._rows.append(row)
        self.epoch += 1

    def compact(self) -> list[tuple[int, int]]:
        """Move the used pages to ``[0, used)``; the page copies to make."""
        used = self.n_pages - len(self._free)
        high = np.nonzero(self.refs[used:])[0] + used
        low = np.nonzero(self.refs[:used] == 0)[0]
        if high.size:
            to = np.arange(self.n_pages, dtype=np.int32)
            to[high] = low
            for row, _, pages in self._seqs.values():
                moved = to[self.table[row, :pages]]
                if not np.array_equal(moved, self.table[row, :pages]):
                    self.table[row, :pages] = moved
                    self.dirty.append((row, 0, pages))
            self.refs[low] = self.refs[high]
            self.refs[high] = 0
            self.epoch += 1
        self._free = list(range(self.n_pages - 1, used - 1, -1))
        return list(zip(high.tolist(), low.tolist()))
