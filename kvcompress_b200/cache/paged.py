"""Paged KV cache held in 4 bits, and the attention that reads it.

No counterpart in the reference, whose int4 compressor
(kvcompress/compressor/quantization_only.py:56-198) only decodes back to dense
tensors: here queries attend the packed codes, sequences of any length share
one pool of pages, and pages are forked, compacted and freed.

Each token's head is quantised in groups of ``group_size`` elements as ``x =
zero + scale * q`` with ``q`` in [-8, 7], ``scale = (max - min) / 15`` and ``zero =
min + 8 * scale`` rounded to float16, ``q`` rounded half to even; a token of a
head costs ``head_dim / 2 + 4 * head_dim / group_size`` bytes each for K and V.
Magnitudes above 65024 are held as 65024; a NaN makes its group NaN.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from functools import partial
from typing import Any, Sequence

import numpy as np
import torch

from kvcompress_b200 import ops
from kvcompress_b200._native import Kv4Layout, Kv4Split, Kv4Step
from kvcompress_b200.cache.pages import PageTable

__all__ = ["CacheStep", "PagedKVCache"]

_CHUNK = 256  # tokens of the smallest item of the attention's split


def _capturing(device: torch.device) -> bool:
    if device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


class _Fence:
    """What the cache itself has put on a stream (a table's update, page copies, a
    step's arrays), for the other streams that use it."""

    __slots__ = ("device", "event", "streams", "bufs")

    def __init__(self, device: torch.device, *bufs: torch.Tensor) -> None:
        self.device, self.bufs = device, bufs  # ``bufs``: memory not to be reused before its uses are done
        with torch.cuda.device(device):
            self.event = torch.cuda.Event()
        self.mark()

    def mark(self) -> None:
        """The work ends here, on the device's current stream."""
        with torch.cuda.device(self.device):
            self.event.record()
        self.streams = {ops._raw_stream(self.device.index)}  # streams that are behind it

    def use(self, stream: int) -> None:
        """Put the raw ``stream``, the device's current one, behind the work."""
        if stream not in self.streams:
            self._join(stream)

    def _join(self, stream: int) -> None:
        # a stream under capture cannot wait for one outside; its graph runs after
        # whatever the program made sure was done before
        if _capturing(self.device):
            return
        cur = torch.cuda.current_stream(self.device)
        cur.wait_event(self.event)
        for buf in self.bufs:
            buf.record_stream(cur)
        self.streams.add(stream)


class _Upload(_Fence):
    """int32 arrays in one device buffer, copied from pinned memory on the
    current stream (torch keeps that until the copy is done).

    Kernels index with these arrays, so on whatever stream one is launched, it
    has to come after the copy, and the buffer must not be reused before it."""

    __slots__ = ("at",)

    def __init__(self, arrays: Sequence[np.ndarray], device: torch.device) -> None:
        if _capturing(device):
            raise RuntimeError("PagedKVCache: a step is planned on its first use, which cannot be captured into a CUDA "
                               "graph; use the step once before")
        host = torch.empty(max(1, sum(a.size for a in arrays)), dtype=torch.int32, pin_memory=True)
        view, n, offsets = host.numpy(), 0, []
        for a in arrays:
            view[n:n + a.size] = a
            offsets.append(n)
            n += a.size
        buf = host.to(device, non_blocking=True)
        super().__init__(device, buf)
        self.at = [buf.data_ptr() + 4 * o for o in offsets]  # the arrays' addresses


@dataclass
class CacheStep:
    """The new tokens, or the queries, of some sequences: made by
    ``PagedKVCache.extend`` / ``view``, used by every layer's ``write`` / ``attend``.

    ``counts[i]`` tokens belong to ``seqs[i]``, the last ones of its
    ``lengths[i]`` cached tokens.  A step is good until a fork, free, truncate
    or compact changes the cache.  Its arrays go to the device on its first use."""

    seqs: list[int]
    counts: list[int]
    lengths: list[int]
    writable: bool
    epoch: int
    cache: Any = field(repr=False)
    meta: _Upload | None = field(default=None, repr=False)  # the arrays that ``desc`` points into
    desc: Kv4Step | None = field(default=None, repr=False)
    splits: dict[tuple[int, int], tuple[list, list]] = field(default_factory=dict, repr=False)

    @property
    def tokens(self) -> int:
        return sum(self.counts)


def _prefix(counts: np.ndarray) -> np.ndarray:
    out = np.zeros(counts.size + 1, dtype=np.int64)
    np.cumsum(counts, out=out[1:])
    return out


_START = 192  # what a CTA's start and end cost, in tokens (about 20 ns each)


def split_chunk(lengths: np.ndarray, copies: int, slots: int, joined: int = 0) -> tuple[int, float]:
    """Tokens of an item so that ``copies`` CTAs an item fill ``slots`` resident
    CTAs evenly, and the cost: of one to four full waves (or no split at all) the
    choice that costs least.  In tokens of a CTA: a wave costs its item and
    ``_START``, joining 200 and a token for every 100 kB of partial results
    (``joined`` bytes an item of every sequence)."""
    longest = int(lengths.max(initial=1))
    total = max(1, int(lengths.sum()))
    best, cost = 0, float("inf")
    for waves in (0, 1, 2, 3, 4):
        chunk = longest if waves == 0 else max(_CHUNK, -(-total * copies // (waves * slots)))
        chunk = -(-chunk // 128) * 128
        items = int(np.maximum(1, -(-lengths // chunk)).sum())
        while waves and chunk < longest and items * copies > waves * slots:
            chunk += max(128, chunk // 32 // 128 * 128)
            items = int(np.maximum(1, -(-lengths // chunk)).sum())
        c = -(-items * copies // slots) * (min(chunk, longest) + _START)
        if items > lengths.size:
            c += 200 + joined * items / lengths.size * 1e-5
        if c < cost:
            best, cost = chunk, c
    return best, cost


def split_items(lengths: np.ndarray, copies: int, slots: int, joined: int, spanning: bool):
    """The attention's items and the blocks that work on them: ``(sequence, first
    token, end, items of each sequence, first item of each block)``.

    Equal pieces of one sequence (``split_chunk``), a block each; or, where blocks
    may span sequences and that costs less: all tokens, in runs of 128, lie in one
    row, which ``slots // copies`` blocks (at least two runs each) cut into equal
    shares, and an item ends where a share or a sequence does.  That wins on
    ragged batches, where equal pieces leave SMs idle (33 sequences of up to 8191
    tokens: 63 against 68 us), and loses where pieces happen to fit (4 x 131072:
    62 against 59 us), since a block with two items starts and ends twice."""
    n = lengths.size
    chunk, cost = split_chunk(lengths, copies, slots, joined)
    start = _prefix(np.maximum(1, -(-lengths // 128)))
    total = int(start[-1])
    blocks = min(slots // copies, -(-total // (_CHUNK // 128)))
    if spanning and blocks > 0 and n * copies < 4 * slots:
        share = -(-total // blocks)
        shares = np.arange(0, total, share)
        cuts = np.unique(np.concatenate((start[:-1], shares)))  # runs at which items begin
        block = np.append(np.searchsorted(cuts, shares), cuts.size)
        if share * 128 + _START * int(np.diff(block).max()) + 200 + joined * cuts.size / n * 1e-5 < cost:
            seq = np.searchsorted(start, cuts, side="right") - 1
            end = np.minimum((np.append(cuts[1:], total) - start[seq]) * 128, lengths[seq])
            return seq, (cuts - start[seq]) * 128, end, np.searchsorted(cuts, start), block
    items = np.maximum(1, -(-lengths // chunk))
    first_item = _prefix(items)
    seq = np.repeat(np.arange(n), items)
    first = (np.arange(int(first_item[-1])) - first_item[seq]) * chunk
    return seq, first, np.minimum(first + chunk, lengths[seq]), first_item, np.arange(int(first_item[-1]) + 1)


class PagedKVCache:
    """K and V of ``n_layers`` layers in 4 bits, in pages of ``page_size`` tokens.

    ``page_size`` is 16, 32, 64, 128 or 256, ``head_dim`` 64 or 128, ``group_size``
    32, 64 or 128 (default ``head_dim``).  ``max_sequences`` sequences of up to
    ``max_tokens`` tokens can live at once (their page table is ``max_sequences *
    max_tokens / page_size`` int32).

    A step of a model::

        step = cache.extend(seqs, [1] * len(seqs))      # room for the new tokens
        for layer in range(n_layers):
            cache.write(layer, k, v, step)
            out = cache.attend(layer, q, step)

    Launches go to the current stream; use a cache from one stream at a time (what
    it puts on the device by itself is ordered across streams, ``write`` and
    ``attend`` are not).  ``write`` and ``attend`` may be captured into a CUDA graph
    once the step has been used outside one; the graph then repeats that step, and
    must not outlive the cache, which keeps the captured steps' arrays.  ``extend``,
    ``compact`` and a step's first use cannot be captured: a decoding loop, whose
    every token is a new step, runs uncaptured.  There is no gradient through a
    cache in 4 bits.

    A step's host work is paid once for all its layers: ``extend`` 13 to 174 us (1 to
    256 sequences), the first ``write`` 75 to 115 us more than the later ones, the
    first ``attend`` 150 to 185.  Sequences with very different numbers of
    queries are best given steps of their own where one of them has a long context
    (a step is split by its largest number of queries; single tokens beside prompts
    are taken apart already).

    How near 4 bits come depends on K's channels: unit normal queries over 8192
    tokens of rotated keys with 8 of 128 channels 8 times as loud are off by 48% with
    one group a head, 42% with groups of 64 and 32% with groups of 32 (by V alone
    10, 9 and 8%).  An orthogonal rotation of K and of the queries before ``write``
    and ``attend`` (a Hadamard matrix over 128 ** 0.5, say) leaves the logits alone and
    spreads the loud channels: 26, 22 and 21%.
    """

    def __init__(self, *, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64,
                 group_size: int | None = None, max_sequences: int = 256, max_tokens: int | None = None,
                 device: torch.device | str = "cuda") -> None:
        self.n_layers, self.n_kv_heads, self.head_dim = int(n_layers), int(n_kv_heads), int(head_dim)
        self.page_size = int(page_size)
        self.group_size = self.head_dim if group_size is None else int(group_size)
        if self.n_layers < 1 or self.n_kv_heads < 1:
            raise ValueError("PagedKVCache: n_layers and n_kv_heads must be positive")
        if self.head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache: head_dim must be 64 or 128, got {head_dim}")
        if self.page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"PagedKVCache: page_size must be 16, 32, 64, 128 or 256, got {page_size}")
        if self.group_size not in (32, 64, 128) or self.head_dim % self.group_size:
            raise ValueError(f"PagedKVCache: group_size must be 32, 64 or 128 and divide head_dim, got {group_size}")
        self.pages = PageTable(n_pages, page_size, max_sequences,
                               int(n_pages) * self.page_size if max_tokens is None else max_tokens)
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedKVCache: kvcompress_b200 runs on CUDA tensors only (got {device})")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self._scale = self.head_dim ** -0.5
        self.page_bytes = ops.kv4_page_bytes(self.n_kv_heads, self.head_dim, self.page_size, self.group_size)
        # (no inference tensors: a cache made in inference mode is updated outside it too)
        with torch.inference_mode(False):
            # zeros: a page's bytes are defined before its first tokens are written
            self.pool = torch.zeros(self.n_layers, self.pages.n_pages, self.page_bytes, dtype=torch.uint8, device=device)
            self.table = torch.zeros(self.pages.table.shape, dtype=torch.int32, device=device)
            self._byte = torch.zeros(1, dtype=torch.uint8, device=device)  # workspaces are empty_like its expansions
        self._shapes: dict[tuple[int, int, int], tuple[int, int, bool]] = {}
        self._fence = _Fence(device, self.pool, self.table)
        self._captured: dict[int, CacheStep] = {}  # steps in graphs, whose arrays have to stay
        self._layers = [self.pool.data_ptr() + i * self.pool.stride(0) for i in range(self.n_layers)]
        self._layout = Kv4Layout(self.table.data_ptr(), self.table.stride(0), self.pages.n_pages, self.n_kv_heads,
                                 self.head_dim, self.page_size, self.group_size)

    # ---- sequences ---------------------------------------------------------

    def add(self) -> int:
        """A new empty sequence's id."""
        return self.pages.add()

    def length(self, seq: int) -> int:
        """Tokens of ``seq`` in the cache."""
        return self.pages.length(seq)

    def free(self, seq: int) -> None:
        """Forget ``seq``; pages that no fork shares become free."""
        self.pages.free(seq)

    def truncate(self, seq: int, length: int) -> None:
        """Drop ``seq``'s tokens from ``length`` on (drafts that were rejected)."""
        self.pages.truncate(seq, length)

    def fork(self, seq: int) -> int:
        """A new sequence that continues ``seq``: it shares the pages, and whichever
        of the two is extended first takes a copy of a partly filled last page."""
        return self.pages.fork(seq)

    def compact(self) -> int:
        """Move the used pages to the pool's start; returns the number of moved pages."""
        self._no_capture("compact")
        moves = self.pages.compact()
        self._copy(moves)
        self._sync()
        return len(moves)

    def memory_used(self) -> int:
        """Bytes of the pages in use, all layers."""
        return (self.pages.n_pages - self.pages.free_pages) * self.page_bytes * self.n_layers

    # ---- steps -----------------------------------------------------------

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> CacheStep:
        """Room for ``counts[i]`` new tokens of ``seqs[i]`` (``RuntimeError`` without
        enough free pages, nothing changed then); the step to write and attend them with."""
        self._no_capture("extend")
        seqs, counts = [int(s) for s in seqs], [int(n) for n in counts]
        self._copy(self.pages.extend(seqs, counts))
        return self._step(seqs, counts, True)

    def view(self, seqs: Sequence[int], counts: Sequence[int]) -> CacheStep:
        """A step that adds nothing: ``counts[i]`` queries over ``seqs[i]`` as it is.
        Under a causal mask they stand at its last ``counts[i]`` positions (queries
        before its first token see nothing).  A sequence may be named twice."""
        seqs, counts = [int(s) for s in seqs], [int(n) for n in counts]
        if len(seqs) != len(counts):
            raise ValueError(f"PagedKVCache.view: {len(seqs)} sequences but {len(counts)} query counts")
        if any(n < 0 for n in counts):
            raise ValueError("PagedKVCache.view: query counts must not be negative")
        return self._step(seqs, counts, False)

    def _step(self, seqs: list[int], counts: list[int], writable: bool) -> CacheStep:
        if sum(counts) > 2 ** 31 - 1:
            raise ValueError("PagedKVCache: too many tokens in one step")
        return CacheStep(seqs, counts, [self.pages.length(s) for s in seqs], writable, self.pages.epoch, self)

    def _prepare(self, step: CacheStep) -> None:
        """Put the step's arrays on the device."""
        # The attention reads the page table before the kernel in front of it has ended,
        # so the table's update must not be that kernel: the copy below has to follow it.
        self._sync()
        n, lengths = np.array(step.counts, dtype=np.int64), np.array(step.lengths, dtype=np.int64)
        rows = np.array([self.pages.row(s) for s in step.seqs], dtype=np.int64)
        halves = np.zeros_like(n)
        if step.writable:  # aligned runs of 8 tokens that the new ones touch
            halves = np.where(n > 0, (lengths - 1) // 8 - (lengths - n) // 8 + 1, 0)
        q_start, half_start = _prefix(n), _prefix(halves)
        half_seq = np.repeat(np.arange(n.size), halves)
        step.meta = _Upload((rows, lengths, q_start, half_seq, half_start), self.device)
        step.desc = Kv4Step(*step.meta.at, int(half_start[-1]), n.size, int(n.max(initial=0)), int(q_start[-1]))

    def _split(self, step: CacheStep, n_q: int, code: int) -> list[tuple[Kv4Split, int, torch.Tensor | None]]:
        got = step.splits.get((n_q, code))
        if got is None:
            plans = self._plan(step, n_q, code)
            got = step.splits[n_q, code] = [p[:3] for p in plans], [p[3] for p in plans]
        stream = ops._raw_stream(self.device.index)
        for up in got[1]:
            up.use(stream)
        return got[0]

    def _plan(self, step: CacheStep, n_q: int, code: int) -> list[tuple]:
        """The step's launches: one, or two where some sequences have many queries
        and others few, which different kernels are for."""
        lengths = np.array(step.lengths, dtype=np.int64)
        counts = np.array(step.counts, dtype=np.int64)
        rows = np.array([self.pages.row(s) for s in step.seqs], dtype=np.int64)
        spans = {n: self._shape(n, n_q, code)[2] for n in set(step.counts) if n}
        plans = []
        for spanning in (False, True):
            if spanning not in spans.values():
                continue
            at = np.array([i for i, n in enumerate(step.counts) if n and spans[n] == spanning], dtype=np.int64)
            most = int(counts[at].max())
            tiles, resident, _ = self._shape(most, n_q, code)
            joined = 8 * int(counts[at].sum()) * n_q * (self.head_dim + 2)
            seq, first, end, start, blocks = split_items(lengths[at], self.n_kv_heads * tiles, resident, joined, spanning)
            items = np.zeros_like(lengths)
            items[at] = np.diff(start)
            table = np.stack((at[seq], first, end, rows[at][seq]), 1)
            up = _Upload((table.reshape(-1), _prefix(items), blocks), self.device)
            split = Kv4Split(*up.at, seq.size, blocks.size - 1, int(items.max()), most)
            nbytes = ops.kv4_attend_workspace(self._layout, split, n_q)
            plans.append((split, nbytes, self._byte.expand(nbytes) if nbytes else None, up))
        return plans

    def _shape(self, max_new: int, n_q: int, code: int) -> tuple[int, int, bool]:
        got = self._shapes.get((max_new, n_q, code))
        if got is None:
            got = self._shapes[max_new, n_q, code] = ops.kv4_attend_shape(self._layout, max_new, n_q, code, self.device)
        return got

    def _check(self, what: str, layer: int, step: CacheStep) -> int:
        if step.cache is not self:
            raise ValueError(f"PagedKVCache.{what}: the step belongs to another cache")
        if step.epoch != self.pages.epoch:
            raise RuntimeError(f"PagedKVCache.{what}: sequences were forked, freed, truncated or compacted since the "
                               "step was made; make it again")
        if not 0 <= layer < self.n_layers:
            raise IndexError(f"PagedKVCache.{what}: layer {layer} of {self.n_layers}")
        if step.meta is None:
            self._prepare(step)
        stream = ops._raw_stream(self.device.index)
        self._fence.use(stream)
        step.meta.use(stream)
        if stream and _capturing(self.device):  # (the default stream, 0, is never captured)
            self._captured[id(step)] = step
        return self._layers[layer]

    # ---- data ---------------------------------------------------------------

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor, step: CacheStep) -> None:
        """Quantise the step's new K and V of ``layer`` into the pages.

        ``key`` / ``value``: ``(tokens, n_kv_heads, head_dim)``, the sequences' tokens
        one after the other, or ``(B, n_kv_heads, T, head_dim)`` when every sequence
        has T new tokens; float32, float16 or bfloat16, any strides with contiguous
        features."""
        pool = self._check("write", layer, step)
        if not step.writable:
            raise ValueError("PagedKVCache.write: a view adds no tokens; use a step from extend()")
        ops.kv4_write(self._layout, step.desc, pool, key, value, self.device)

    def attend(self, layer: int, query: torch.Tensor, step: CacheStep, *, causal: bool = True,
               scale: float | None = None) -> torch.Tensor:
        """Attention of the step's queries over their sequences' cached tokens.

        ``query``: ``(tokens, n_heads, head_dim)`` or ``(B, n_heads, T, head_dim)``,
        ``n_heads`` a multiple of ``n_kv_heads`` (consecutive query heads share a KV
        head); the result has its shape and dtype.  ``causal``: a query sees the
        tokens up to its own position, otherwise all cached tokens of its sequence;
        one that sees none gets zeros.  ``scale`` defaults to ``head_dim ** -0.5``."""
        pool = self._check("attend", layer, step)
        return ops.kv4_attend(self._layout, step.desc, partial(self._split, step), pool, query, causal=causal,
                              scale=self._scale if scale is None else float(scale), device=self.device)

    def read(self, seq: int, *, layers: Sequence[int] | None = None, t0: int = 0, t1: int | None = None,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """Tokens ``[t0, t1)`` of ``seq`` decoded: K and V, each ``(layers, n_kv_heads,
        t1 - t0, head_dim)``.  ``k[i]``, ``v[i]`` are the cells a ``KVCompressor`` takes.
        ``layers`` (default all) is a range of consecutive layers."""
        n = self.pages.length(seq)
        t0, t1 = int(t0), n if t1 is None else int(t1)
        if not 0 <= t0 <= t1 <= n:
            raise ValueError(f"PagedKVCache.read: bad token range [{t0}, {t1}) of {n}")
        pick = list(range(self.n_layers)) if layers is None else [int(i) for i in layers]
        if pick and (pick != list(range(pick[0], pick[0] + len(pick))) or pick[0] < 0 or pick[-1] >= self.n_layers):
            raise ValueError(f"PagedKVCache.read: layers must be consecutive and within {self.n_layers}, got {pick}")
        self._sync()
        return ops.kv4_read(self._layout, self._layers[pick[0]] if pick else self._layers[0], self.pool.stride(0),
                            len(pick), self.pages.row(seq), t0, t1, dtype, self.device)

    # ---- internals ---------------------------------------------------------

    def _no_capture(self, what: str) -> None:
        if _capturing(self.device):
            raise RuntimeError(f"PagedKVCache.{what}: not possible inside a CUDA graph")

    def _copy(self, pairs: list[tuple[int, int]]) -> None:
        if pairs:
            self._fence.use(ops._raw_stream(self.device.index))
            ops.copy_pages(self.pool, [s for s, _ in pairs], [d for _, d in pairs])
            self._fence.mark()

    def _sync(self) -> None:
        """Bring the device's page table up to the host's."""
        self._fence.use(ops._raw_stream(self.device.index))
        dirty = self.pages.dirty
        if not dirty:
            return
        self._no_capture("read, write or attend after the page table has changed")
        width = self.pages.max_pages
        at = np.concatenate([np.arange(r * width + a, r * width + b) for r, a, b in dirty])
        if len(dirty) > 1 and at.size > len(dirty):  # (the same entry twice gets the same page twice)
            at = np.unique(at)
        host = torch.empty(2, at.size, dtype=torch.int64, pin_memory=True)
        host[0] = torch.from_numpy(at)
        host[1] = torch.from_numpy(self.pages.table.reshape(-1)[at].astype(np.int64))
        dev = host.to(self.device, non_blocking=True)
        self.table.view(-1).index_copy_(0, dev[0], dev[1].to(torch.int32))
        dirty.clear()
        self._fence.mark()
