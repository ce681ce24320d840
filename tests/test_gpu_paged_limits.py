"""The paged 4-bit KV cache at the limits of what it accepts: the longest sequences, far value scales, the most
columns, other modes of torch, memory used on several streams."""

from __future__ import annotations

import gc

import pytest
import torch
from test_gpu_paged import BF16, FP16, FP32, attention, cells, check_attend, held, make, queries, read_equal

from kvcompress_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, nq", [(BF16, 1), (BF16, 16), (FP16, 64), (FP32, 1)])
def test_the_longest_sequence(dtype, nq):
    """2^31 - 300 tokens (the limit is 2^31 - 257) whose table row names the same three pages over and over.  Positions of
    tokens past the last one do not fit in 32 bits: none may be looked up in the table.

    The want: every position of the pages counts as often as the table names it.  Tolerance, of the largest value: the
    products' accumulators drop up to 2^-23 of themselves at each of a warp's additions, about 2^31 / 16 / (296 * 4) =
    113k of them to a sum that grows evenly (half of that counts: 7e-3); the kernel for many queries adds 2^31 / 16 /
    148 times (907k), in float32 accumulators of the same kind (5.4e-2)."""
    n, page = 2 ** 31 - 300, 256
    c = make(1, 64, 64, page, n, 1, pages=3)
    s = c.add()
    k, v = cells(3 * page, 1, 64, dtype)
    c.write(0, k, v, c.extend([s], [3 * page]))
    c.pages._seqs[s][1:] = [n, -(-n // page)]
    c.pages.table[0] = torch.arange(c.pages.max_pages).remainder(3).numpy()
    c.table.copy_(torch.from_numpy(c.pages.table))
    q = queries(nq, 4, 64, dtype, size=0.1)
    got = c.attend(0, q, c.view([s], [nq]), causal=False).double()
    times = torch.full((3 * page,), float(n // (3 * page)), dtype=torch.float64, device="cuda")
    times[:n % (3 * page)] += 1
    k, v = held(k, 64)[:, 0], held(v, 64)[:, 0]
    p = torch.softmax(torch.einsum("nhd,td->nht", q.double(), k) / 8 + times.log(), -1)
    want = torch.einsum("nht,td->nhd", p, v)
    tol = (5.4e-2 if nq >= 16 else 7e-3) + torch.finfo(dtype).eps / 2
    assert (got - want).abs().max() <= tol * v.abs().max()
    assert ops.device_error() == 0


# ---- value scales that lie far apart -----------------------------------------

# How far a group of an output may be off, relative to that group's own norm over all rows.  16-bit outputs: half a step of
# their type (bf16 3.9e-3, fp16 4.9e-4), which over many elements averages below its maximum, and the weights' float16
# half step (4.9e-4), which independent weights average too: their maxima together for bf16, 6e-4 for fp16 (the mean of the two
# squared is 3.4e-4).  float32: logits of sum |q k| <= 5 or so from two-term queries (22 bits) and float32 sums,
# 5 (2^-22 + 2^-21) = 3.6e-6, two-term weights 2^-22.
GROUP_TOL = {BF16: 4.4e-3, FP16: 6e-4, FP32: 4e-6}


def group_errors(c, q, s, k, v, rows=slice(None)):
    got = c.attend(0, q, c.view([s], [q.shape[0]]))
    want, _ = attention(q, held(k, c.group_size), held(v, c.group_size), True, c.head_dim ** -0.5)
    got, want = (x.double()[rows].unflatten(-1, (-1, c.group_size)) for x in (got, want))
    return ((got - want) ** 2).sum((0, 1, 3)).sqrt() / (want ** 2).sum((0, 1, 3)).sqrt()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d, group", [(64, 32), (128, 64), (128, 32)])
@pytest.mark.parametrize("nq", [1, 7, 40])
@pytest.mark.parametrize("far", [12, 20])
def test_quiet_groups_beside_loud_ones(dtype, d, group, nq, far):
    """Every second group's values are 2^12 or 2^20 times as large as the others'."""
    c = make(1, d, group, 64, 2048, 1)
    s = c.add()
    k, v = cells(2000, 1, d, FP32)
    up = 13 if far == 20 else 6
    v = v * torch.where(torch.arange(d, device="cuda") // group % 2 == 0, 2.0 ** up, 2.0 ** (up - far))
    k, v = k.to(dtype), v.to(dtype)
    c.write(0, k, v, c.extend([s], [2000]))
    off = group_errors(c, queries(nq, 4, d, dtype, size=0.5), s, k, v)
    assert (off <= GROUP_TOL[dtype]).all(), off


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d, group", [(64, 64), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("heads", [1, 2, 3])
def test_loud_tokens_that_only_later_queries_see(dtype, d, group, heads):
    """The last four tokens' values are 2^20 times as large: the first four queries' results must not know."""
    c = make(1, d, group, 64, 2048, 1)
    s = c.add()
    k, v = cells(1500, 1, d, FP32)
    v[:-4] *= 2.0 ** -7
    v[-4:] *= 2.0 ** 13
    k, v = k.to(dtype), v.to(dtype)
    c.write(0, k, v, c.extend([s], [1500]))
    q = queries(8, heads, d, dtype, size=0.5)
    for rows in (slice(0, 4), slice(4, 8)):
        off = group_errors(c, q, s, k, v, rows)
        assert (off <= GROUP_TOL[dtype]).all(), (rows, off)


@pytest.mark.parametrize("d, group", [(64, 64), (128, 128), (128, 32)])
@pytest.mark.parametrize("nq", [1, 6])
def test_a_loud_token_of_next_to_no_weight(d, group, nq):
    """One token's values are 2^18 times as large, and its weight e^-25: the others' weights keep their bits."""
    c = make(1, d, group, 64, 2048, 1)
    s = c.add()
    k, v = cells(1500, 1, d, FP32)
    v = v * 2.0 ** -8
    q = queries(nq, 4, d, FP32, size=0.02)
    q[..., -1] = 4.0
    k[..., -1] = 0.0
    k[100, 0, -1] = -6.25 * d ** 0.5
    v[100] *= 2.0 ** 18
    c.write(0, k, v, c.extend([s], [1500]))
    off = group_errors(c, q, s, k, v)
    assert (off <= GROUP_TOL[FP32]).all(), off


# ---- more columns or items than a grid's third extent ---------------------------


def same_for_all(q, k, v, group):
    """Each query (n, H, d) over all of k and v (T, 1, d), in float64."""
    k, v = held(k, group)[:, 0], held(v, group)[:, 0]
    return torch.softmax(q.double() @ k.T * q.shape[-1] ** -0.5, -1) @ v


def test_more_than_65535_tiles_of_float32_columns():
    c = make(1, 64, 64, 16, 64, 1)
    s = c.add()
    k, v = cells(40, 1, 64, FP32)
    c.write(0, k, v, c.extend([s], [40]))
    q = queries(1025, 1024, 64, FP32)  # 1049600 columns in tiles of 16
    got = c.attend(0, q, c.view([s], [1025]), causal=False)
    want = same_for_all(q, k, v, 64)
    assert (got - want).norm() <= 1e-5 * want.norm()
    assert (got - want).abs().max() <= 1e-4 * v.abs().max()


def test_more_than_65535_items_of_many_columns():
    c = make(1, 64, 64, 16, 64, 1)
    s = c.add()
    k, v = cells(20, 1, 64, BF16)
    c.write(0, k, v, c.extend([s], [20]))
    n = 65600
    q = queries(n, 64, 64, BF16)  # 64 columns each: the kernel for many queries
    got = c.attend(0, q, c.view([s] * n, [1] * n))
    want = same_for_all(q, k, v, 64)
    assert (got - want).norm() <= 5e-3 * want.norm()
    assert (got - want).abs().max() <= 2 ** -7 * v.abs().max()


# ---- other modes of torch ----------------------------------------------------


@pytest.mark.parametrize("made, used", [(True, False), (False, True), (True, True)])
def test_inference_mode(made, used):
    """A cache made in inference mode is used outside it, and the other way round."""
    k, v = cells(70, 2, 64, BF16)
    q = queries(3, 4, 64, BF16)
    with torch.inference_mode(made):
        c = make(2, 64, pages=64)
        a = c.add()
        c.write(0, k[:30], v[:30], c.extend([a], [30]))
    with torch.inference_mode(used):
        b = c.fork(a)
        c.write(0, k[30:], v[30:], c.extend([b], [40]))
        out = c.attend(0, q, c.view([b], [3]))
        c.free(a)
        c.compact()
        assert torch.equal(out, c.attend(0, q, c.view([b], [3])))
    with torch.inference_mode(made):
        c.truncate(b, 50)
        c.write(0, k[50:], v[50:], c.extend([b], [20]))
        check_attend(c, q, c.view([b], [3]), [(k, v)])
        read_equal(c, b, k, v)


def test_copied_pages_and_autograd():
    for many in (False, True):
        pool = torch.randn(2, 4, 8, device="cuda")
        w = torch.ones_like(pool).requires_grad_()
        want = pool.clone()
        want[:, 1] = want[:, 0]
        y = (pool * w).sum()
        ops.copy_pages(list(pool.unbind(0)) if many else pool, [0], [1])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        assert torch.equal(pool, want)
        pool.requires_grad_()
        for x in (pool, pool * 1):
            with pytest.raises(RuntimeError, match="gradient"):
                ops.copy_pages(list(x.unbind(0)) if many else x, [2], [3])
        assert torch.equal(pool, want)
        with torch.no_grad():
            ops.copy_pages(list(pool.unbind(0)) if many else pool, [2], [3])
            want[:, 3] = want[:, 2]
        assert torch.equal(pool, want)
        with torch.inference_mode():
            x = pool * 1
            ops.copy_pages(list(x.unbind(0)) if many else x, [0], [2])
            want[:, 2] = want[:, 0]
        assert torch.equal(x, want)


# ---- memory used on several streams ---------------------------------------------


def test_a_dropped_caches_memory_is_kept_for_another_streams_work():
    c = make(2, 64, 64, 64, 64 * 4000, 1, dirty=False)
    s = c.add()
    k, v = cells(3000, 2, 64, BF16)
    q = queries(1, 4, 64, BF16)
    c.write(0, k, v, c.extend([s], [3000]))
    step = c.view([s], [1])
    want = c.attend(0, q, step)
    torch.cuda.synchronize()
    at, shape = c.pool.data_ptr(), c.pool.shape
    assert c.pool.numel() > 20 << 20  # a block of its own, which the allocator would hand out again at once
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # about half a second, longer than the collection below
        got = c.attend(0, q, step)
    del c, step
    gc.collect()
    new = torch.empty(shape, dtype=torch.uint8, device="cuda")
    assert not side.query()
    assert new.data_ptr() != at
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ---- roundings -------------------------------------------------------------------


def loud_cells(n, d, dtype, by, off):
    """K with d / 16 channels `by` times as loud, half of them shifted by `off`."""
    g = torch.Generator(device="cuda").manual_seed(3)
    size, shift = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
    at = torch.randperm(d, generator=g, device="cuda")[:d // 16]
    size[at] = by
    shift[at[::2]] = off
    k = torch.randn(n, 1, d, generator=g, device="cuda") * size + shift
    return k.to(dtype), torch.randn(n, 1, d, generator=g, device="cuda").to(dtype)


# (not float32 with far offsets: its own rounding of logits of hundreds dominates there)
@pytest.mark.parametrize("dtype, by, off", [(t, by, off) for t in (BF16, FP16, FP32)
                                            for by, off in ((8, 4), (20, 4), (8, 60), (8, 200)) if t != FP32 or off == 4])
@pytest.mark.parametrize("d, group", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("nq", [2, 8, 60])
def test_roundings_are_those_that_are_stated(dtype, by, off, d, group, nq):
    """The norm of the error over 1500 tokens, against the roundings that each path is to have.

    A value rounded to m bits (half a step 2^-m of its power of two) is off by 2^-m / sqrt 3 of that power in the mean square,
    0.72 of which is the mean relative error of evenly spread mantissas: bf16 (m = 8) 1.63e-3, float16 (m = 11) 2.0e-4.
    Outputs, weights and values (one float16 rounding each at most) are independent: sqrt 3 2.0e-4 = 3.5e-4 for float16
    outputs, 1.65e-3 for bf16.  Where held K is rounded to float16 (bfloat16 queries of more than 48 columns), a logit is
    off by 2^-11 / sqrt 3 of each |q k| at most, added as squares; an independent error of the logits changes the result
    by as much.  float32 queries: 22-bit terms and float32 sums of logits up to 20."""
    c = make(1, d, group, 64, 2048, 1)
    s = c.add()
    k, v = loud_cells(1500, d, dtype, by, off)
    c.write(0, k, v, c.extend([s], [1500]))
    q = queries(nq, 4, d, dtype, size=1.0)
    got = c.attend(0, q, c.view([s], [nq]), causal=False).double()
    kh = held(k, group)
    want, _ = attention(q, kh, held(v, group), False, d ** -0.5)
    tol = {BF16: 2e-3, FP16: 4e-4, FP32: 2e-6}[dtype]
    if dtype == BF16 and nq * 4 > 48:
        squares = torch.einsum("nhd,td->nht", q.double() ** 2, kh[:, 0] ** 2).mean().item()
        tol = (tol ** 2 + squares / d * 2.0 ** -22 / 3) ** 0.5
    err = ((got - want).norm() / want.norm()).item()
    assert err <= tol, (err, tol)


@pytest.mark.parametrize("nq", [1, 48, 49, 100])
def test_a_bad_page_is_reported_by_both_kernels(nq):
    c = make(1, 64, 64, 16, 128, 2)
    s = c.add()
    k, v = cells(120, 1, 64, BF16)
    assert ops.device_error() == 0
    c.write(0, k, v, c.extend([s], [120]))
    c.table[c.pages.row(s), 1] = c.pages.n_pages
    c.attend(0, queries(nq, 1, 64, BF16), c.view([s], [nq]))
    assert ops.device_error() == 401
    c.table[c.pages.row(s), 1] = -1
    c.attend(0, queries(nq, 1, 64, BF16), c.view([s], [nq]))
    assert ops.device_error() == 401
    assert ops.device_error() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d, group", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)])
def test_columns_on_both_sides_of_the_kernels_limit(dtype, d, group):
    c = make(2, d, group, 32, 1024, 3)
    seqs = [c.add() for _ in range(3)]
    lens = [700, 33, 1000]
    k, v = cells(sum(lens), 2, d, dtype)
    c.write(0, k, v, c.extend(seqs, lens))
    kv = list(zip(k.split(lens), v.split(lens)))
    for counts in ([16, 16, 16], [17, 17, 17], [15, 16, 17], [32, 33, 30], [1, 17, 33], [100, 33, 1]):  # of 3 columns each
        for causal in (True, False):
            check_attend(c, queries(sum(counts), 6, d, dtype), c.view(seqs, counts), kv, causal)


@pytest.mark.parametrize("d, group", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("nq, lens", [(26, [3000]), (200, [4000]), (150, [2500, 800, 64, 63])])
def test_repeated_float16_calls_give_the_same_bits(d, group, nq, lens):
    """Tiles in two terms, whose codes two sets of warps read: one that came too late or too early would show."""
    c = make(4, d, group, 32, 4096, len(lens), pages=300)
    seqs = [c.add() for _ in lens]
    k, v = cells(sum(lens), 4, d, FP16)
    c.write(0, k, v, c.extend(seqs, lens))
    step = c.view(seqs, [nq] * len(lens))
    q = queries(nq * len(lens), 16, d, FP16)
    out = check_attend(c, q, step, list(zip(k.split(lens), v.split(lens))))
    assert not torch.stack([(c.attend(0, q, step) != out).any() for _ in range(60)]).any()
    assert ops.device_error() == 0
