"""The paged 4-bit KV cache against its definition in 64 bits.

What a token's head is held as is defined exactly (``held``), so ``read`` is
compared bit for bit.  ``attend`` is compared with the attention over those
values in float64 under the bound of ``bound``.
"""

from __future__ import annotations

import gc
import math

import numpy as np
import pytest
import torch

from kvcompress_b200 import PagedKVCache, build_compressor, ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)]  # head_dim, group_size


def held(x, group):
    """The values a head (..., d) is held as, in float64."""
    g = x.double().clamp(-65024.0, 65024.0).unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).float().half().double()
    zero = (lo + 8 * scale).float().half().double()
    q = torch.where(scale > 0, ((g - zero) / torch.where(scale > 0, scale, 1.0)).round(), 0.0).clamp(-8, 7)
    return (zero + scale * q).flatten(-2)


def attention(q, k, v, causal, scale):
    """(n, Hq, d) queries over (T, Hkv, d) in float64; the largest sum of |q_j k_j| scale."""
    n, hq, d = q.shape
    t, hkv = k.shape[:2]
    if t == 0 or n == 0:
        return torch.zeros(n, hq, d, dtype=torch.float64, device=q.device), 0.0
    k = k.repeat_interleave(hq // hkv, 1)
    s = torch.einsum("nhd,thd->hnt", q.double(), k) * scale
    size = (torch.einsum("nhd,thd->hnt", q.double().abs(), k.abs()) * abs(scale)).nan_to_num().max().item()
    if causal:
        at = torch.arange(t, device=q.device)
        s = s.masked_fill(at > t - n + torch.arange(n, device=q.device)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    w = w.masked_fill(s == -math.inf, 0.0)
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    vis = w.transpose(0, 1)  # (n, h, t)
    out = torch.einsum("nht,thd->nhd", vis, torch.nan_to_num(v, nan=0.0).repeat_interleave(hq // hkv, 1))
    bad = torch.isnan(v).any(-1).repeat_interleave(hq // hkv, 1)  # (t, h)
    seen = (s != -math.inf).transpose(0, 1)
    out[(seen & bad.t()[None]).any(-1) | torch.isnan(s).any(-1).t()] = math.nan
    return out, size


def bound(want, vals, size, dtype):
    """How far an output may be off: the logits' error first.  16-bit queries: products of operands rounded by at
    most u = 2^-12 (a held value to float16), summed in float32: |dS| <= size (2^-12 + 2^-18); float32: the queries'
    two float16 terms carry 22 bits, |dS| <= size 2^-18 with the sums.  Weights change by a factor within
    exp(2 dS) and are rounded to float16 (2^-12; float32: two terms, 2^-20 with the sums), against values of
    magnitude at most max|v|, and values are rounded to float16 once more (2^-12); then the output's own half step."""
    u = 2.0 ** -18 if dtype == FP32 else 2.0 ** -12 + 2.0 ** -18
    w = 2.0 ** -18 if dtype == FP32 else 2.0 ** -11
    vmax = vals.abs().nan_to_num().max().item() if vals.numel() else 0.0
    return torch.finfo(dtype).eps / 2 * want.abs() + vmax * (math.expm1(2 * size * u) + w) + 1e-30


def cells(n, h, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn(n, h, d, generator=g, device="cuda")
    k[..., : d // 16] = k[..., : d // 16] * 3 + 1
    return k.to(dtype), torch.randn(n, h, d, generator=g, device="cuda").to(dtype)


def queries(n, h, d, dtype, seed=1, size=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, h, d, generator=g, device="cuda") * size).to(dtype)


def make(h=2, d=128, group=None, page=16, tokens=512, seqs=8, layers=1, pages=None, dirty=True):
    c = PagedKVCache(n_layers=layers, n_pages=pages or seqs * -(-tokens // page), n_kv_heads=h, head_dim=d,
                     page_size=page, group_size=group, max_sequences=seqs, max_tokens=tokens)
    if dirty:
        c.pool.fill_(255)  # NaN parameters wherever nothing is written
    return c


def check_attend(c, q, step, kv, causal=True, scale=None, layer=0):
    out = c.attend(layer, q, step, causal=causal, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    flat = out if q.dim() == 3 else out.transpose(1, 2).flatten(0, 1)
    qf = q if q.dim() == 3 else q.transpose(1, 2).flatten(0, 1)
    at = 0
    for n, (k, v) in zip(step.counts, kv):
        k, v = held(k, c.group_size), held(v, c.group_size)
        want, size = attention(qf[at:at + n], k, v, causal, c.head_dim ** -0.5 if scale is None else scale)
        got = flat[at:at + n].double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        if fine.any():
            off = (got - want).abs()[fine]
            tol = bound(want, v, size, q.dtype)[fine]
            assert (off <= tol).all(), (off / tol).max().item()
            # and far closer on the whole than the worst case
            rel = (got - want)[fine].norm() / want[fine].norm().clamp_min(1e-30)
            assert rel <= {FP32: 1e-5, FP16: 1e-3, BF16: 5e-3}[q.dtype], rel
        at += n
    return out


def read_equal(c, seq, k, v, layer=0, dtype=None):
    dtype = dtype or k.dtype
    ko, vo = c.read(seq, layers=[layer], dtype=dtype)
    for got, x in ((ko[0], k), (vo[0], v)):
        want = held(x, c.group_size).float().to(dtype).transpose(0, 1)
        assert got.shape == want.shape
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


# ---- write and read ------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d, group", SHAPES)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_read_gives_what_is_defined(dtype, d, group, page):
    c = make(3, d, group, page, 700, 2)
    a, b = c.add(), c.add()
    ka, va = cells(333, 3, d, dtype)
    kb, vb = cells(91, 3, d, dtype, 7)
    at = 0
    for n in (1, 1, 6, 7, 16, 9, 33, 260):  # halves and units entered and left at every phase
        step = c.extend([a], [n])
        c.write(0, ka[at:at + n], va[at:at + n], step)
        at += n
    for i in range(0, 91, 13):
        c.write(0, kb[i:i + 13], vb[i:i + 13], c.extend([b], [13]))
    assert at == 333
    read_equal(c, a, ka, va)
    read_equal(c, b, kb, vb)
    read_equal(c, b, kb, vb, dtype=FP32)
    k, v = c.read(a, t0=5, t1=322, dtype=FP16)
    assert torch.equal(k[0].float(), held(ka, group).float().half().float()[5:322].transpose(0, 1))
    assert torch.equal(v[0].float(), held(va, group).float().half().float()[5:322].transpose(0, 1))
    assert c.read(a, t0=7, t1=7)[0].shape == (1, 3, 0, d)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_special_values(dtype):
    d = 128
    k, v = cells(40, 2, d, dtype)
    big = 6e4 if dtype == FP16 else 3e38
    k[0], v[0] = 0.0, -2.5  # constant groups: scale 0
    k[1, 0, 5], v[1, 1, 77] = math.nan, math.nan
    k[2, 0, 0], v[2, 0, 1] = math.inf, -math.inf
    k[3, 1], v[3, 1] = big, 1e-7  # beyond the held range (clamped), below float16's smallest step
    k[4, :, ::2], v[4, :, ::2] = big, -big
    k[4, :, 1::2] = -big
    k[5] = torch.arange(d, device="cuda").remainder(31).to(dtype) / 2  # 0 .. 15 in halves: scale 1, exact ties
    v[5] = k[5] - 7.5
    k[6] = k[6].to(dtype) * 1e-3 + 100  # an offset that is large against the spread
    for group in (128, 64, 32):
        c = make(2, d, group)
        s = c.add()
        c.write(0, k, v, c.extend([s], [40]))
        read_equal(c, s, k, v)


def test_ties_are_decided_exactly():
    """x = zero + (n + 1/2) scale and its float32 neighbours, for scales of all 11 bits."""
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = 512
    scale = (1 + torch.rand(rows, 1, generator=g, device="cuda")).half().float()
    lo = (torch.randn(rows, 1, generator=g, device="cuda") * 4).half().float()
    n = torch.randint(0, 15, (rows, 64), generator=g, device="cuda") + 0.5
    x = lo + n * scale
    x = torch.where(torch.rand(rows, 64, generator=g, device="cuda") < 0.5, x, torch.nextafter(x, x + 1))
    x[:, 0:1], x[:, 1:2] = lo, lo + 15 * scale
    c = make(1, 64, 64, 64, 512, 1)
    s = c.add()
    x = x.view(rows, 1, 64)
    c.write(0, x, -x, c.extend([s], [rows]))
    read_equal(c, s, x, -x)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides_and_layouts_of_inputs(dtype):
    d, h, b, t = 128, 3, 2, 21
    big_k, big_v = cells(b * t, 2 * h + 1, 2 * d, dtype)
    for off in (0, 1):  # the odd offset leaves no alignment
        k, v = big_k[:, 1::2, off:off + d], big_v[:, 1::2, off:off + d]
        c = make(h, d)
        seqs = [c.add(), c.add()]
        c.write(0, k, v, c.extend(seqs, [t, t]))
        for i, s in enumerate(seqs):
            read_equal(c, s, k[i * t:(i + 1) * t], v[i * t:(i + 1) * t])
        c4 = make(h, d)
        seqs = [c4.add(), c4.add()]
        k4, v4 = (x.unflatten(0, (b, t)).transpose(1, 2) for x in (k, v))  # (B, h, T, d)
        c4.write(0, k4, v4, c4.extend(seqs, [t, t]))
        for i, s in enumerate(seqs):
            read_equal(c4, s, k[i * t:(i + 1) * t], v[i * t:(i + 1) * t])
        c4.write(0, k4.contiguous(), v4, c4._step(seqs, [t, t], True))  # K and V of different strides


def test_a_write_touches_only_its_tokens():
    c = make(2, 128, 128, 16, 512, 4)
    a, b = c.add(), c.add()
    k, v = cells(50, 2, 128, BF16)
    c.write(0, k[:25], v[:25], c.extend([a], [25]))
    step = c.extend([a, b], [3, 0])
    before = c.pool.clone()
    c.write(0, k[25:28], v[25:28], step)
    changed = (c.pool != before).nonzero()[:, 1].unique().tolist()
    assert changed == [c.pages.pages(a)[1]]
    assert int((c.pool != before).sum()) <= 3 * 2 * (128 + 8)
    read_equal(c, a, k[:28], v[:28])


# ---- attention ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d, group", SHAPES)
@pytest.mark.parametrize("hq, hkv", [(8, 1), (7, 7), (28, 4), (24, 1), (64, 2)])
def test_single_tokens(dtype, d, group, hq, hkv):
    lens = [1, 2, 15, 16, 17, 31, 33, 300, 257, 511]
    c = make(hkv, d, group, 16, 512, len(lens))
    seqs = [c.add() for _ in lens]
    k, v = cells(sum(lens), hkv, d, dtype)
    c.write(0, k, v, c.extend(seqs, lens))
    kv = list(zip(k.split(lens), v.split(lens)))
    check_attend(c, queries(len(lens), hq, d, dtype), c.view(seqs, [1] * len(lens)), kv)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d, group, page", [(64, 64, 16), (64, 32, 64), (128, 128, 64), (128, 64, 32), (128, 32, 256)])
@pytest.mark.parametrize("counts", [[2, 3, 1, 5], [8, 0, 1, 8], [33, 1, 70, 129], [5, 128, 200, 256]])
def test_several_queries(dtype, causal, d, group, page, counts):
    lens = [700, 1, 129, 256]  # the second sequence is shorter than its queries: rows that see nothing
    hq, hkv = 6, 2
    c = make(hkv, d, group, page, 1024, 4)
    seqs = [c.add() for _ in lens]
    k, v = cells(sum(lens), hkv, d, dtype)
    c.write(0, k, v, c.extend(seqs, lens))
    kv = list(zip(k.split(lens), v.split(lens)))
    check_attend(c, queries(sum(counts), hq, d, dtype), c.view(seqs, counts), kv, causal)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_empty_sequences_and_empty_steps(dtype):
    c = make(2, 128)
    a, b = c.add(), c.add()
    k, v = cells(9, 2, 128, dtype)
    c.write(0, k, v, c.extend([a], [9]))
    for causal in (True, False):
        q = queries(5, 4, 128, dtype)
        out = check_attend(c, q, c.view([a, b], [2, 3]), [(k, v), (k[:0], v[:0])], causal)
        assert not out[2:].any()
        assert c.attend(0, q[:0], c.view([a, b], [0, 0]), causal=causal).shape == (0, 4, 128)
        assert c.attend(0, q[:0], c.view([], []), causal=causal).shape == (0, 4, 128)
    c.write(0, k[:0], v[:0], c.extend([a], [0]))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nq", [3, 40, 300])
def test_nan_reaches_only_the_queries_that_see_it(dtype, nq):
    c = make(2, 128, 128, 32, 512, 2)
    s = c.add()
    k, v = cells(400, 2, 128, dtype)
    k[398, 0, 3], v[397, 1, 9] = math.nan, math.nan  # seen by the last queries of one head each
    c.write(0, k, v, c.extend([s], [400]))
    q = queries(nq, 4, 128, dtype)
    out = check_attend(c, q, c.view([s], [nq]), [(k, v)])
    assert not torch.isnan(out[:nq - 3]).any() and torch.isnan(out[-1]).all()
    v[10, 0, 0] = math.inf  # held as the largest value
    q[0, 1, 5] = math.nan  # a query's own NaN stays its own
    c.truncate(s, 0)
    c.write(0, k[:390], v[:390], c.extend([s], [390]))
    out = c.attend(0, q, c.view([s], [nq]))
    assert torch.isnan(out[0, 1]).all() == (nq <= 390) and not torch.isnan(out[1:]).any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("nq", [1, 64])
def test_loud_tokens_and_far_scales(dtype, nq):
    """Maxima that grow along the cache, value scales of many magnitudes, a sink that takes most weight."""
    c = make(1, 128, 128, 64, 2048, 1)
    s = c.add()
    k, v = cells(2000, 1, 128, dtype)
    k = (k * torch.linspace(0.05, 3, 2000, device="cuda")[:, None, None]).to(dtype)
    v = (v * torch.logspace(-3, 2, 2000, device="cuda")[torch.randperm(2000, device="cuda")][:, None, None]).to(dtype)
    k[0] = 4
    c.write(0, k, v, c.extend([s], [2000]))
    q = queries(nq, 4, 128, dtype)
    check_attend(c, q, c.view([s], [nq]), [(k, v)])
    check_attend(c, q, c.view([s], [nq]), [(k, v)], scale=0.01)
    check_attend(c, q, c.view([s], [nq]), [(k, v)], scale=-0.05)
    check_attend(c, q, c.view([s], [nq]), [(k, v)], scale=0.0)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("mag", [1e-30, 1e-6, 1e3])
def test_query_magnitudes(dtype, mag):
    if dtype == FP16 and mag == 1e-30:
        mag = 1e-7
    c = make(1, 64, 64, 16, 256, 1)
    s = c.add()
    k, v = cells(200, 1, 64, dtype)
    c.write(0, k, v, c.extend([s], [200]))
    for nq in (2, 100):
        q = queries(nq, 2, 64, FP32, size=1.0)
        q[0, 0] = 0
        q[0, 1, 3:] *= 1e-4
        q = (q * mag).to(dtype)
        check_attend(c, q, c.view([s], [nq]), [(k, v)], scale=0.02 / max(mag, 1e-30))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("t", [1, 5, 40])
def test_query_strides_and_layouts(dtype, t):
    d, hq, hkv, b = 128, 6, 2, 3
    c = make(hkv, d)
    seqs = [c.add() for _ in range(b)]
    lens = [50, 130, 77]
    k, v = cells(sum(lens), hkv, d, dtype)
    c.write(0, k, v, c.extend(seqs, lens))
    kv = list(zip(k.split(lens), v.split(lens)))
    step = c.view(seqs, [t] * b)
    big = queries(b * t, 2 * hq, 2 * d, dtype)
    want = check_attend(c, big[:, ::2, :d].contiguous(), step, kv)
    for off in (0, 1):
        q = torch.empty_like(big)
        q[:, ::2, off:off + d] = big[:, ::2, :d]
        q = q[:, ::2, off:off + d]
        assert torch.equal(c.attend(0, q, step), want)
        q4 = q.unflatten(0, (b, t)).transpose(1, 2)
        assert torch.equal(c.attend(0, q4, step).transpose(1, 2).flatten(0, 1), want)
        assert torch.equal(c.attend(0, q4.contiguous(), step).transpose(1, 2).flatten(0, 1), want)


@pytest.mark.parametrize("lens, nq, hkv", [([40000], 1, 2), ([9000, 1, 30000, 500], 2, 1), ([20011], 64, 1)])
def test_long_caches_are_split_and_joined(lens, nq, hkv):
    c = make(hkv, 128, 128, 64, 40960, len(lens), pages=sum(-(-n // 64) for n in lens))
    seqs = [c.add() for _ in lens]
    for dtype in (BF16, FP32):
        for s in seqs:
            c.truncate(s, 0)
        k, v = cells(sum(lens), hkv, 128, dtype)
        c.write(0, k, v, c.extend(seqs, lens))
        kv = list(zip(k.split(lens), v.split(lens)))
        q = queries(nq * len(lens), 4, 128, dtype, size=0.1)
        step = c.view(seqs, [nq] * len(lens))
        out = check_attend(c, q, step, kv)
        assert torch.equal(out, c.attend(0, q, step))  # the joining order is fixed


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d, group", SHAPES)
@pytest.mark.parametrize("nq, lens", [(1, [6000, 5000, 17]), (4, [3000, 2999]), (200, [4000])])
def test_repeated_calls_give_the_same_bits(dtype, d, group, nq, lens):
    """Rings of codes are refilled while they are read: a call that read too late would differ."""
    c = make(4, d, group, 32, 8192, len(lens), pages=500)
    seqs = [c.add() for _ in lens]
    k, v = cells(sum(lens), 4, d, dtype)
    c.write(0, k, v, c.extend(seqs, lens))
    step = c.view(seqs, [nq] * len(lens))
    q = queries(nq * len(lens), 16, d, dtype)
    out = c.attend(0, q, step)
    assert not torch.stack([(c.attend(0, q, step) != out).any() for _ in range(40)]).any()


def test_offsets_beyond_32_bits():
    """Pages past 4 GiB of the pool and past 2^31 elements of the output."""
    page, h = 256, 8
    n_pages = (9 << 30) // 2 // (h * 16 * 2176) + 2  # 4.5 GiB a layer
    c = PagedKVCache(n_layers=2, n_pages=n_pages, n_kv_heads=h, head_dim=128, page_size=page, max_sequences=2,
                     max_tokens=page * n_pages)
    low, s = c.add(), c.add()
    c.extend([low], [page * (n_pages - 3)])
    k, v = cells(600, h, 128, BF16)
    step = c.extend([s], [600])
    assert min(c.pages.pages(s)) * c.page_bytes > 1 << 32
    c.write(1, k, v, step)
    read_equal(c, s, k, v, layer=1)
    check_attend(c, queries(1, 8, 128, BF16), c.view([s], [1]), [(k, v)], layer=1)
    check_attend(c, queries(100, 8, 128, BF16), c.view([s], [100]), [(k, v)], layer=1)
    n = c.compact()
    assert n == 0
    c.free(low)
    c.compact()
    assert sorted(c.pages.pages(s)) == [0, 1, 2]
    read_equal(c, s, k, v, layer=1)


# ---- pages -------------------------------------------------------------------


def test_forks_diverge_and_share():
    c = make(2, 128, 64, 32, 512, 6, layers=3)
    a = c.add()
    k, v = cells(300, 2, 128, BF16)
    extra = [cells(40, 2, 128, BF16, 10 + i) for i in range(3)]

    def put(seq_kv):
        step = c.extend(list(seq_kv), [x[0].shape[0] for x in seq_kv.values()])
        for layer in range(3):
            c.write(layer, torch.cat([x[0] for x in seq_kv.values()]) + layer,
                    torch.cat([x[1] for x in seq_kv.values()]) + layer, step)

    put({a: (k[:100], v[:100])})
    free = c.pages.free_pages
    b, d = c.fork(a), c.fork(a)
    assert c.pages.free_pages == free
    put({a: extra[0], b: extra[1], d: extra[2]})  # one call: two copies of the shared last page
    want = {s: (torch.cat([k[:100], e[0]]), torch.cat([v[:100], e[1]])) for s, e in zip((a, b, d), extra)}
    c.truncate(b, 64)
    want[b] = (k[:64], v[:64])
    c.free(a)
    del want[a]
    moved = c.compact()
    assert moved > 0
    used = c.pages.n_pages - c.pages.free_pages
    assert c.memory_used() == used * c.page_bytes * 3
    for s, (x, y) in want.items():
        assert max(c.pages.pages(s)) < used
        for layer in range(3):
            read_equal(c, s, x + layer, y + layer, layer=layer)
        check_attend(c, queries(2, 4, 128, BF16), c.view([s], [2]), [(x + 1, y + 1)], layer=1)
    step = c.view([d, b, d], [1, 2, 3])  # the same sequence twice
    check_attend(c, queries(6, 4, 128, BF16), step, [want[d], want[b], want[d]])


@pytest.mark.parametrize("dtype, inner", [(BF16, (16, 2, 64)), (torch.uint8, (37,)), (FP32, (3, 3)), (torch.float8_e4m3fn, (20,)),
                                          (torch.int64, (1000, 5))])
def test_copy_pages(dtype, inner):
    pool = torch.randint(0, 100, (3, 50) + inner, device="cuda").to(dtype)
    raw = pool.view(torch.uint8).clone()
    src, dst = [0, 0, 49, 7], [1, 48, 2, 30]
    ops.copy_pages(pool, src, dst)
    raw[:, dst] = raw[:, src]
    assert torch.equal(pool.view(torch.uint8), raw)
    some = [pool[0], pool[2]]
    ops.copy_pages(some, [5], [6])
    raw[0, 6], raw[2, 6] = raw[0, 5], raw[2, 5]
    assert torch.equal(pool.view(torch.uint8), raw)
    ops.copy_pages(pool, [], [])
    ops.copy_pages([], [], [])
    ops.copy_pages(torch.empty(3, 5, 0, device="cuda"), [0], [1])
    ops.copy_pages(torch.empty(0, 5, 2, device="cuda"), [0], [1])
    for far in (1 << 31, -(1 << 40)):
        with pytest.raises(ValueError, match="out of range"):
            ops.copy_pages(pool, [0], [far])
    for twice in (torch.tensor([2, 2]), [torch.tensor(2), torch.tensor(2)], np.array([2, 2])):
        with pytest.raises(ValueError, match="written twice"):
            ops.copy_pages(pool, [0, 1], twice)
    with pytest.raises(TypeError):
        ops.copy_pages(pool, [0.0], [1])
    for bad in (([0], [50]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [])):
        with pytest.raises(ValueError):
            ops.copy_pages(pool, *bad)
    with pytest.raises(ValueError):
        ops.copy_pages(pool.transpose(0, 1), [0], [1])
    assert torch.equal(pool.view(torch.uint8), raw)


def test_copy_pages_many_pairs_and_pools():
    pool = torch.randint(0, 1 << 30, (70, 5000, 4), device="cuda", dtype=torch.int32)
    want = pool.clone()
    order = torch.randperm(5000).tolist()
    src, dst = order[:2400], order[2400:4800]
    ops.copy_pages(pool, src, dst)
    want[:, dst] = want[:, src]
    assert torch.equal(pool, want)
    pools = list(pool.unbind(0))
    ops.copy_pages(pools, dst[:3], src[:3])
    want[:, src[:3]] = want[:, dst[:3]]
    assert torch.equal(pool, want)


# ---- how a program uses them -----------------------------------------------------


def test_refusals():
    c = make(2, 128, layers=2)
    s = c.add()
    k, v = cells(4, 2, 128, BF16)
    step = c.extend([s], [4])
    with pytest.raises(ValueError):
        c.write(0, k[:3], v[:3], step)
    with pytest.raises(ValueError):
        c.write(0, k, v.half(), step)
    with pytest.raises(ValueError):
        c.write(0, k[:, :1], v[:, :1], step)
    with pytest.raises(ValueError):
        c.write(0, k[..., :64], v[..., :64], step)
    with pytest.raises(ValueError):
        c.write(0, *(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)), step)
    with pytest.raises(TypeError):
        c.write(0, k.int(), v.int(), step)
    with pytest.raises(RuntimeError):
        c.write(0, k.cpu(), v.cpu(), step)
    with pytest.raises(IndexError):
        c.write(2, k, v, step)
    c.write(0, k, v, step)
    q = queries(4, 4, 128, BF16)
    with pytest.raises(ValueError, match="no multiple"):
        c.attend(0, q[:, :3], step)
    with pytest.raises(ValueError):
        c.attend(0, q[:3], step)
    with pytest.raises(ValueError):
        c.attend(0, q[0], step)
    with pytest.raises(TypeError):
        c.attend(0, q.double(), step)
    with pytest.raises(RuntimeError, match="gradient"):
        c.attend(0, q.clone().requires_grad_(), step)
    with torch.no_grad():
        c.attend(0, q.clone().requires_grad_(), step)
    with pytest.raises(ValueError, match="another cache"):
        make(2, 128).attend(0, q, step)
    view = c.view([s], [4])
    with pytest.raises(ValueError, match="view"):
        c.write(0, k, v, view)
    other = c.fork(s)
    for old in (step, view):
        with pytest.raises(RuntimeError, match="make it again"):
            c.attend(0, q, old)
    with pytest.raises(RuntimeError, match="make it again"):
        c.write(0, k, v, step)
    with pytest.raises(ValueError):
        c.read(other, t0=0, t1=5)
    with pytest.raises(ValueError):
        c.read(other, layers=[0, 2])
    with pytest.raises(TypeError):
        c.read(other, dtype=torch.int8)
    with pytest.raises(ValueError):
        c.view([s], [-1])
    c.free(other)
    with pytest.raises(KeyError):
        c.read(other)


def test_captured_steps_replay():
    """write and attend in CUDA graphs: replays see new inputs, two graphs keep apart on two streams."""
    c = make(2, 128, 128, 64, 20000, 4, layers=2, pages=700)
    seqs = [c.add(), c.add()]
    lens = [12000, 9000]
    k, v = cells(sum(lens), 2, 128, BF16)
    before = c.extend(seqs, lens)
    for layer in range(2):
        c.write(layer, k, v, before)
    step = c.extend(seqs, [1, 1])
    graphs = []
    for layer in range(2):
        kn, vn = cells(2, 2, 128, BF16, 20 + layer)
        q = queries(2, 8, 128, BF16, 30 + layer)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            c.write(layer, kn, vn, step)
            c.attend(layer, q, step)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                c.write(layer, kn, vn, step)
                out = c.attend(layer, q, step)
        torch.cuda.current_stream().wait_stream(stream)
        graphs.append((g, stream, kn, vn, q, out))
    for rep in range(3):
        for layer, (g, stream, kn, vn, q, out) in enumerate(graphs):
            a, b = cells(2, 2, 128, BF16, 40 + 2 * rep + layer)
            kn.copy_(a), vn.copy_(b), q.copy_(queries(2, 8, 128, BF16, 50 + 2 * rep + layer))
        torch.cuda.synchronize()
        for g, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for layer, (g, stream, kn, vn, q, out) in enumerate(graphs):
            want = c.attend(layer, q, step)
            assert torch.equal(out, want)
            kv = [(torch.cat([x, kn[i:i + 1]]), torch.cat([y, vn[i:i + 1]]))
                  for i, (x, y) in enumerate(zip(k.split(lens), v.split(lens)))]
            check_attend(c, q, step, kv, layer=layer)


def test_a_new_step_is_not_planned_inside_a_graph():
    c = make(2, 128)
    s = c.add()
    k, v = cells(40, 2, 128, BF16)
    q = queries(1, 4, 128, BF16)
    c.write(0, k, v, c.extend([s], [40]))
    step = c.view([s], [1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="use the step once before"):
            c.attend(0, q, step)
        with pytest.raises(RuntimeError, match="use the step once before|inside a CUDA graph"):
            c.write(0, k[:1], v[:1], c.extend([s], [1]))
        q.add_(0)
    c.truncate(s, 40)
    check_attend(c, q, c.view([s], [1]), [(k, v)])


def test_a_captured_step_may_be_dropped():
    """The graph's step arrays stay, whatever the allocator hands out afterwards."""
    c = make(2, 128, 128, 64, 20000, 2, pages=400)
    s = c.add()
    k, v = cells(9000, 2, 128, BF16)
    q = queries(3, 4, 128, BF16)
    c.write(0, k, v, c.extend([s], [9000]))
    step = c.view([s], [3])
    want = c.attend(0, q, step)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.attend(0, q, step)
        with pytest.raises(RuntimeError, match="inside a CUDA graph"):
            c.extend([s], [1])
        with pytest.raises(RuntimeError, match="inside a CUDA graph"):
            c.compact()
    assert c.length(s) == 9000
    del step
    gc.collect()
    torch.cuda.synchronize()
    # in range whatever the old arrays' bytes become: all zeros
    junk = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 8, 64, 128, 512, 1024) for _ in range(40)]
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert len(junk) == 240 and ops.device_error() == 0


def test_page_copies_are_ordered_before_another_streams_use():
    """extend's copy of a shared page waits on a busy stream; the step is used on another one."""
    c = make(2, 128, 128, 64, 256, 2)
    s = c.add()
    k, v = cells(100, 2, 128, BF16)
    c.write(0, k[:99], v[:99], c.extend([s], [99]))
    f = c.fork(s)
    q = queries(1, 4, 128, BF16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(20_000_000)  # about 10 ms on the current stream
    step = c.extend([f], [1])
    with torch.cuda.stream(side):
        c.write(0, k[99:], v[99:], step)
        out = c.attend(0, q, step)
    torch.cuda.synchronize()
    assert torch.equal(out, c.attend(0, q, step))
    check_attend(c, q, step, [(k, v)])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [6, 50])
def test_queries_whose_strides_overlap(dtype, n):
    c = make(2, 128, 128, 64, 1024, 2)
    s = c.add()
    k, v = cells(500, 2, 128, dtype)
    c.write(0, k, v, c.extend([s], [500]))
    base = queries(n + 4, 1, 128, dtype).flatten()
    for q in (base.as_strided((n, 4, 128), (1, 64, 1)), base[:128].expand(n, 4, 128), base.as_strided((n, 4, 128), (2, 2, 1))):
        out = check_attend(c, q, c.view([s], [n]), [(k, v)])
        assert torch.equal(out, c.attend(0, q.contiguous(), c.view([s], [n])))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("counts", [[1, 300, 1, 0, 40, 1, 2], [2000, 1, 1, 1, 1, 1, 1]])
def test_prompts_and_single_tokens_in_one_step(dtype, counts):
    lens = [9000, 310, 1, 50, 700, 5000, 20]
    lens[0] = max(lens[0], counts[0])
    c = make(2, 128, 128, 64, 16384, 7, pages=400)
    seqs = [c.add() for _ in lens]
    k, v = cells(sum(lens), 2, 128, dtype)
    c.write(0, k, v, c.extend(seqs, lens))
    kv = list(zip(k.split(lens), v.split(lens)))
    q = queries(sum(counts), 8, 128, dtype, size=0.1)
    for causal in (True, False):
        check_attend(c, q, c.view(seqs, counts), kv, causal)


def test_another_stream():
    c = make(2, 128, 128, 16, 4096, 2)
    s = c.add()
    k, v = cells(3000, 2, 128, BF16)
    q = queries(1, 4, 128, BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.write(0, k, v, c.extend([s], [3000]))
        out = c.attend(0, q, c.view([s], [1]))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, c.attend(0, q, c.view([s], [1])))
    check_attend(c, q, c.view([s], [1]), [(k, v)])


def test_a_step_used_on_another_stream_waits_for_its_arrays():
    """The step's stream is busy when another one uses the step, and the step is
    dropped and its memory overwritten while that one still works."""
    c = make(2, 128, 128, 64, 40960, 2, pages=700)
    s = c.add()
    k, v = cells(30000, 2, 128, BF16)
    q = queries(1, 4, 128, BF16)
    c.write(0, k, v, c.extend([s], [30000]))
    want = c.attend(0, q, c.view([s], [1]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(20_000_000)  # about 10 ms on the current stream
    step = c.view([s], [1])
    with torch.cuda.stream(side):
        outs = [c.attend(0, q, step) for _ in range(50)]
    del step
    for _ in range(20):
        torch.full((64,), 1 << 20, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert ops.device_error() == 0


def test_a_bad_page_is_reported_and_skipped():
    c = make(1, 64, 64, 16, 64, 2)
    s = c.add()
    k, v = cells(40, 1, 64, BF16)
    assert ops.device_error() == 0
    step = c.extend([s], [40])
    c.write(0, k, v, step)
    c.table[c.pages.row(s), 1] = c.pages.n_pages
    for nq in (1, 40):
        c.attend(0, queries(nq, 1, 64, BF16), c.view([s], [nq]))
        assert ops.device_error() == 401
    c.read(s)
    assert ops.device_error() == 401
    c.write(0, k, v, step)
    assert ops.device_error() == 401
    assert ops.device_error() == 0


def test_serving_run():
    """Prompts in chunks, decoding, drafts and their rejection, a fork, an eviction through a compressor and back."""
    d, hq, hkv, layers = 128, 8, 2, 2
    c = make(hkv, d, 128, 16, 2048, 6, layers=layers, pages=200)
    seqs = {c.add(): [cells(0, hkv, d, BF16)] * layers for _ in range(3)}

    def step(counts, seed, view=False):
        names = list(counts)
        st = c.extend(names, list(counts.values()))
        n = sum(counts.values())
        for layer in range(layers):
            k, v = cells(n, hkv, d, BF16, seed + layer)
            c.write(layer, k, v, st)
            for s, a, b in zip(names, k.split(list(counts.values())), v.split(list(counts.values()))):
                old = seqs[s][layer]
                seqs[s] = list(seqs[s])
                seqs[s][layer] = (torch.cat([old[0], a]), torch.cat([old[1], b]))
            check_attend(c, queries(n, hq, d, BF16, seed), st, [seqs[s][layer] for s in names], layer=layer)

    a, b, e = seqs
    step({a: 200, b: 77}, 1)
    step({a: 130, b: 1, e: 40}, 10)
    for i in range(20):
        step({a: 1, b: 1, e: 1}, 100 + i)
    f = c.fork(b)
    seqs[f] = list(seqs[b])
    step({b: 5, f: 5, e: 1}, 200)
    c.truncate(b, c.length(b) - 3)
    seqs[b] = [(k[:-3], v[:-3]) for k, v in seqs[b]]
    c.free(a)
    del seqs[a]
    c.compact()
    step({e: 1, f: 1, b: 1}, 300)
    # an idle sequence leaves through a compressor and comes back
    k, v = c.read(e)
    comp = build_compressor("int8")
    pay = [comp.compress(k[i], v[i]) for i in range(layers)]
    c.free(e)
    del seqs[e]
    g = c.add()
    back = c.extend([g], [k.shape[2]])
    seqs[g] = []
    for layer, (kp, vp) in enumerate(pay):
        kd, vd = comp.decompress(kp, vp)
        c.write(layer, kd[None], vd[None], back)
        seqs[g].append((kd.transpose(0, 1), vd.transpose(0, 1)))
    step({b: 1, f: 1, g: 1}, 400)
    for s, kv in seqs.items():
        for layer in range(layers):
            read_equal(c, s, *kv[layer], layer=layer)
    assert ops.device_error() == 0
