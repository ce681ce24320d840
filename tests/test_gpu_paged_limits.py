"""The paged 4-bit KV cache at the limits of what it accepts: the longest sequences, far value scales, the most
columns, other modes of torch, memory used on several streams."""

from __future__ import annotations

import pytest
import torch
from test_gpu_paged import BF16, FP32, attention, cells, held, make, queries

from kvcompress_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, nq", [(BF16, 1), (BF16, 16), (FP32, 1)])
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
    tol = (5.4e-2 if nq == 16 else 7e-3) + torch.finfo(dtype).eps / 2
    assert (got - want).abs().max() <= tol * v.abs().max()
    assert ops.device_error() == 0
