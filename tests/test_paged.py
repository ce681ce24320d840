"""Page accounting of the paged cache, and what its entry points refuse (CPU)."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest
import torch

from kvcompress_b200 import PagedKVCache, ops
from kvcompress_b200._native import KVC, Kv4Layout, Kv4Split, Kv4Step, lib
from kvcompress_b200.cache.pages import PageTable
from kvcompress_b200.cache.paged import split_chunk, split_items


def _check(t: PageTable, tokens: dict, content: dict) -> None:
    """``content[page][slot]`` is the token each page slot holds: every sequence reads its own tokens back."""
    refs = np.zeros(t.n_pages, dtype=int)
    for seq, toks in tokens.items():
        pages = t.pages(seq)
        assert t.length(seq) == len(toks) and len(pages) == -(-len(toks) // t.page_size)
        for p in pages:
            refs[p] += 1
        for i, tok in enumerate(toks):
            assert content[pages[i // t.page_size]][i % t.page_size] == tok
    assert (refs == t.refs).all() and t.free_pages == int((refs == 0).sum())
    assert sorted(t._free) == np.nonzero(refs == 0)[0].tolist()


def test_random_operations_keep_every_sequence():
    rng = random.Random(3)
    t = PageTable(40, 16, 8, 160)
    tokens, content, fresh = {}, {p: [None] * 16 for p in range(40)}, 0
    for _ in range(1500):
        op = rng.choice(("add", "extend", "extend", "extend", "fork", "free", "truncate", "compact"))
        seqs = list(tokens)
        try:
            if op == "add":
                tokens[t.add()] = []
            elif op == "extend" and seqs:
                some = rng.sample(seqs, rng.randint(1, len(seqs)))
                n = [rng.choice((0, 1, 1, 5, 16, 30)) for _ in some]
                before = (t.table.copy(), t.refs.copy(), list(t._free))
                try:
                    copies = t.extend(some, n)
                except (RuntimeError, ValueError):  # refused: nothing changed
                    assert (t.table == before[0]).all() and (t.refs == before[1]).all() and t._free == before[2]
                    raise
                for src, dst in copies:
                    content[dst] = list(content[src])
                for s, k in zip(some, n):
                    pages = t.pages(s)
                    for _ in range(k):
                        i, fresh = len(tokens[s]), fresh + 1
                        assert t.refs[pages[i // 16]] == 1  # a page that takes tokens is its sequence's own
                        content[pages[i // 16]][i % 16] = fresh
                        tokens[s].append(fresh)
            elif op == "fork" and seqs:
                s = rng.choice(seqs)
                tokens[t.fork(s)] = list(tokens[s])
            elif op == "free" and seqs:
                s = rng.choice(seqs)
                t.free(s)
                del tokens[s]
            elif op == "truncate" and seqs:
                s = rng.choice(seqs)
                k = rng.randint(0, len(tokens[s]))
                t.truncate(s, k)
                del tokens[s][k:]
            elif op == "compact":
                moves = t.compact()
                src, dst = [a for a, _ in moves], [b for _, b in moves]
                assert len(set(dst)) == len(dst) and set(src).isdisjoint(dst)
                for a, b in moves:
                    content[b] = list(content[a])
                used = 40 - t.free_pages
                assert all(p < used for s in tokens for p in t.pages(s))
        except (RuntimeError, ValueError):
            pass
        _check(t, tokens, content)


def test_both_forks_extended_at_once_copy_a_shared_page_once():
    t = PageTable(8, 16, 4, 64)
    a = t.add()
    t.extend([a], [20])
    b = t.fork(a)
    shared = t.pages(a)[1]
    copies = t.extend([a, b], [1, 1])
    assert copies == [(shared, t.pages(a)[1])] and t.pages(b)[1] == shared
    assert t.pages(a)[0] == t.pages(b)[0]
    assert t.extend([a, b], [1, 1]) == []
    c = t.fork(b)
    assert t.extend([c], [0]) == []  # no new token, no copy


def test_full_last_page_is_not_copied():
    t = PageTable(8, 16, 4, 64)
    a = t.add()
    t.extend([a], [32])
    b = t.fork(a)
    assert t.extend([b], [1]) == []
    assert t.pages(a) == t.pages(b)[:2] and len(t.pages(b)) == 3


def test_page_table_refusals():
    t = PageTable(4, 16, 2, 48)
    a = t.add()
    with pytest.raises(ValueError, match="exceed max_tokens"):
        t.extend([a], [49])
    with pytest.raises(ValueError, match="twice"):
        t.extend([a, a], [1, 1])
    with pytest.raises(ValueError, match="negative"):
        t.extend([a], [-1])
    with pytest.raises(ValueError, match="counts"):
        t.extend([a], [])
    with pytest.raises(KeyError):
        t.extend([7], [1])
    t.extend([a], [48])
    b = t.add()
    with pytest.raises(RuntimeError, match="out of pages"):
        t.extend([b], [17])
    with pytest.raises(RuntimeError, match="in use"):
        t.add()
    with pytest.raises(RuntimeError, match="in use"):
        t.fork(a)
    with pytest.raises(ValueError, match="cannot keep"):
        t.truncate(a, 49)
    t.free(b)
    with pytest.raises(KeyError):
        t.free(b)
    for bad in ((0, 16, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0)):
        with pytest.raises(ValueError):
            PageTable(*bad)


def test_split_chunk_covers_and_bounds():
    for lens, copies in (([1], 1), ([0, 0], 8), ([17], 4), ([32768] * 8, 8), ([131072] * 4, 4), ([5] * 999, 64),
                         ([2 ** 31 - 300], 1), (list(range(0, 8191, 253)), 8)):
        chunk, _ = split_chunk(np.array(lens, dtype=np.int64), copies, 296)
        assert chunk % 128 == 0 and 128 <= chunk < 2 ** 31


@pytest.mark.parametrize("spanning", [True, False])
@pytest.mark.parametrize("lens, copies", [([1], 1), ([0, 0], 8), ([17], 4), ([32768] * 8, 8), ([131072] * 4, 4), ([5] * 999, 64),
                                          ([2 ** 31 - 300], 1), (list(range(0, 8191, 253)), 8), ([0, 700, 0, 1], 2),
                                          ([128] * 7 + [100000], 3), ([300] * 50, 500)])
def test_items_cover_every_sequence_once(lens, copies, spanning):
    n = np.array(lens, dtype=np.int64)
    seq, first, end, start, blocks = split_items(n, copies, 444, 1000, spanning)
    assert start[0] == 0 and start[-1] == seq.size and blocks[0] == 0 and blocks[-1] == seq.size
    assert (np.diff(blocks) >= 1).all() and blocks.size - 1 <= max(444, seq.size)
    for i, m in enumerate(lens):
        at = 0
        assert start[i + 1] > start[i]
        for j in range(start[i], start[i + 1]):
            assert seq[j] == i and first[j] == at and first[j] % 128 == 0 and end[j] <= m
            at = end[j]
        assert at == m


@pytest.mark.parametrize("kw, err", [
    (dict(head_dim=96), ValueError), (dict(page_size=48), ValueError), (dict(group_size=16), ValueError),
    (dict(head_dim=64, group_size=128), ValueError), (dict(n_layers=0), ValueError), (dict(n_kv_heads=0), ValueError),
    (dict(n_pages=0), ValueError), (dict(device="cpu"), RuntimeError)])
def test_cache_refuses(kw, err):
    args = dict(n_layers=1, n_pages=4, n_kv_heads=2, head_dim=128)
    args.update(kw)
    with pytest.raises(err):
        PagedKVCache(**args)


def test_copy_pages_refusals():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.copy_pages(torch.zeros(2, 4, 8), [0], [1])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.copy_pages([torch.zeros(4, 8)], [0], [1])
    with pytest.raises(ValueError):
        ops.copy_pages(torch.zeros(4), [0], [1])


def _abi():
    table = (1 << 20)  # an address that no refused call reads
    layout = Kv4Layout(table, 4, 8, 2, 128, 16, 128)
    step = Kv4Step(table, table, table, table, table, 1, 1, 1, 1)
    split = Kv4Split(table, table, table, 1, 1, 1, 1)
    return layout, step, split, table


@pytest.mark.parametrize("field, value", [("head_dim", 96), ("page_size", 24), ("page_size", 512), ("group_size", 8),
                                          ("n_kv", 0), ("n_pages", 0), ("table_stride", 0), ("table", None)])
def test_abi_refuses_bad_layouts(field, value):
    layout, step, split, p = _abi()
    setattr(layout, field, value)
    L = lib()
    assert L.kvc_kv4_write(layout, step, p, p, p, KVC.BF16, 0, 256, 128, 1, None) < 0
    assert L.kvc_kv4_read(layout, p, 0, 1, 0, 0, 1, KVC.BF16, p, p, None) < 0
    assert L.kvc_kv4_attend(layout, step, split, p, 2, p, 0, 256, 128, p, 0, 256, 128, 1, KVC.BF16, 1, 1.0, None, 0,
                            None) < 0
    assert L.kvc_last_error()


@pytest.mark.parametrize("field", ["rows", "kv_len", "q_start", "half_seq", "half_start"])
def test_abi_refuses_missing_step_arrays(field):
    layout, step, split, p = _abi()
    setattr(step, field, None)
    L = lib()
    assert L.kvc_kv4_write(layout, step, p, p, p, KVC.BF16, 0, 256, 128, 1, None) == KVC.ERR_ARG
    if not field.startswith("half"):
        assert L.kvc_kv4_attend(layout, step, split, p, 2, p, 0, 256, 128, p, 0, 256, 128, 1, KVC.BF16, 1, 1.0, None, 0,
                                None) == KVC.ERR_ARG


def test_abi_refuses_bad_arguments():
    layout, step, split, p = _abi()
    L = lib()
    assert L.kvc_kv4_write(layout, step, p, None, p, KVC.BF16, 0, 256, 128, 1, None) == KVC.ERR_ARG
    assert L.kvc_kv4_write(layout, step, p, p, p, KVC.F64, 0, 256, 128, 1, None) < 0
    assert L.kvc_kv4_write(layout, step, p + 8, p, p, KVC.BF16, 0, 256, 128, 1, None) < 0
    assert L.kvc_kv4_read(layout, p, 0, 1, 0, 2, 1, KVC.BF16, p, p, None) < 0
    assert L.kvc_kv4_read(layout, p, 0, 1, 0, 0, 65, KVC.BF16, p, p, None) < 0  # past the table's row
    assert L.kvc_kv4_read(layout, p, 0, 1, 0, 0, 1, KVC.BF16, p, p + 4, None) < 0
    bad = dict(n_q=3), dict(dtype=KVC.F64), dict(q=None), dict(pool=p + 4)
    for kw in bad:
        a = dict(n_q=2, dtype=KVC.BF16, q=p, pool=p)
        a.update(kw)
        assert L.kvc_kv4_attend(layout, step, split, a["pool"], a["n_q"], a["q"], 0, 256, 128, p, 0, 256, 128, 1,
                                a["dtype"], 1, 1.0, None, 0, None) < 0
    one = (ctypes.c_void_p * 1)(p)
    i32 = (ctypes.c_int32 * 2)(0, 9)
    assert L.kvc_copy_pages(1, one, 4, 16, 1, i32, (ctypes.c_int32 * 1)(4), None) < 0  # dst out of range
    assert L.kvc_copy_pages(1, one, 4, 16, 2, i32, (ctypes.c_int32 * 2)(1, 2), None) < 0  # src out of range
    assert L.kvc_copy_pages(65, one, 4, 16, 1, i32, (ctypes.c_int32 * 1)(1), None) < 0
    assert L.kvc_copy_pages(1, one, 4, 16, 0, None, None, None) == KVC.OK
    assert L.kvc_kv4_page_bytes(8, 128, 64, 128) == 8 * 4 * 2176


