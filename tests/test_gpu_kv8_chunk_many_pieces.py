"""A chunk so long that every block of the grid takes several pieces of work of hundreds of microseconds each: the one that lists
them waits for whole pieces, far longer than a tile. Rows picked over the chunk against 64 bits, with test_gpu_kv8_chunk's bound."""
import math

import pytest
import torch

from larder_b200 import ops

import serve_ref as ref
from test_gpu_kv8_chunk import BF, cache, close, i32, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,n,hq,hk", [(32768, 8192, 32, 8), (16384, 16384, 16, 8)])
def test_many_long_pieces_a_block(L, n, hq, hk):
    d = 128
    pages, scales, table = cache([L], hk, 64, d)
    q = queries(hq, n, d, BF)
    rows = sorted({0, 1, n // 3, n // 2 - 1, n - 1} | set(range(37, n, 611)))
    want, a = (torch.empty(hq, len(rows), d, dtype=torch.float64, device="cuda") for _ in range(2))
    hidden = torch.arange(L, device="cuda") > torch.tensor([L - n + r for r in rows], device="cuda")[:, None]
    for h in range(hk):
        k, v = (ref.held(pages, scales, table[0], L, i, h) for i in (0, 1))
        for x in range(h * (hq // hk), (h + 1) * (hq // hk)):
            s = (q[0, x, rows].double() @ k.T * d ** -0.5).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1)
            want[x], a[x] = p @ v, p @ v.abs()
    for _ in range(3):
        out = torch.full_like(q, float("nan"))
        ops.kv8_attend_packed(q, pages, scales, table, i32([L]), i32([0, n]), d ** -0.5, out=out)
        assert ops.status() == 0 and torch.isfinite(out).all()
        close(out[:, :, rows], want, a, BF)
