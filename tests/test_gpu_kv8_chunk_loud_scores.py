"""Chunk attention where scores are so large that fp32 numbers of their size lie far apart. Scores here are one product of a query's
one dim with a key's code, so that a key's score is that product rounded a few times, 2^-22 of it in all: keys whose codes differ
stay in their order, and a row's largest one, 1/14 above the next, has all the weight. Its output is then that key's value:
off by its own rounding and by that of the weight's product, |err| <= (u + 2^-11) |v|."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref
from test_gpu_kv8_chunk import BF, HF, F, cache, close, expect, i32, queries, starts

pytestmark = pytest.mark.gpu


def loud(lens, counts, hq, hk, page, d, sign):
    """Pages, queries of one dim each, and for every row the position of the key with the largest score of those it sees."""
    pages, scales, table = cache(lens, hk, page, d, spread=1.0)
    raw, g = pages.view(torch.uint8), torch.Generator().manual_seed(1)
    T = sum(counts)
    q = torch.zeros(1, hq, T, d, device="cuda")
    best = torch.zeros(hq, T, dtype=torch.long)
    at = 0
    for b, (L, n) in enumerate(zip(lens, counts)):
        # codes below the top in no order, the top once for each dim, in a key that every row sees
        k = torch.randint(1, 0x7D, (hk, L, d), generator=g, dtype=torch.uint8)
        top = torch.randint(0, max(L - n, 0) + 1, (hk, d), generator=g)
        k.scatter_(1, top[:, None], 0x7E)
        if sign < 0:
            k |= 0x80
        for h in range(hk):
            for p in range(L):
                raw[int(table[b, p // page]), 0, h, p % page] = k[h, p].cuda()
        scales[table[b, :-(-L // page)].long(), 0] = 2.0 ** -9
        for x in range(hq):
            dim = torch.randint(0, d, (n,), generator=g)
            q[0, x, torch.arange(at, at + n), dim.cuda()] = 1.0 + torch.randint(0, 64, (n,), generator=g).cuda() / 64
            best[x, at:at + n] = top[x // (hq // hk)][dim]
        at += n
    return pages, scales, table, q, best


def values(pages, scales, table, lens, counts, G, best):
    """The values at `best`, fp64 [Hq, T, D]."""
    want = torch.zeros(*best.shape, pages.shape[4], dtype=torch.float64, device="cuda")
    for x in range(best.shape[0]):
        at = 0
        for b, n in enumerate(counts):
            want[x, at:at + n] = ref.held(pages, scales, table[b], lens[b], 1, x // G)[best[x, at:at + n].cuda()]
            at += n
    return want


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens,counts,hq,hk", [([70, 300], [30, 141], 4, 2), ([1900], [200], 2, 1)])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_score_takes_the_row(lens, counts, hq, hk, d, dtype, sign):
    pages, scales, table, q, best = loud(lens, counts, hq, hk, 16, d, sign)
    q = q.to(dtype)
    want = values(pages, scales, table, lens, counts, hq // hk, best)
    for e in (10, 16, 19, 20, 21, 22, 23, 24, 25, 27, 30, 40, 60, 100):
        got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), sign * 1.2345 * 2.0 ** e)
        err = (got[0].double() - want).abs()
        bad = ~(err <= (ref.UNIT[dtype] + 2.0 ** -11) * want.abs() + (2.0 ** -25 if dtype == HF else 0))
        assert not bad.any(), (e, int(bad.any(-1).sum()), got[0][bad][:4], want[bad][:4])
    assert ops.status() == 0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_values_scales_far_apart(d, dtype):
    """The largest score's value may lie in a page whose scale is 2^87 below the others'. (Scores are 100 and more apart.)"""
    lens, counts = [70, 300, 1900], [30, 141, 50]
    pages, scales, table, q, best = loud(lens, counts, 4, 2, 16, d, 1)
    scales[table[:, 1].long(), 1] = 2.0 ** -95
    want = values(pages, scales, table, lens, counts, 2, best)
    assert (want.abs().amax(-1) < 2.0 ** -80).any()
    for e in (12, 19, 20, 21, 24, 27, 40, 100):
        got = ops.kv8_attend_packed(q.to(dtype), pages, scales, table, i32(lens), i32(starts(counts)), 1.2345 * 2.0 ** e)
        err = (got[0].double() - want).abs()
        assert (err <= (ref.UNIT[dtype] + 2.0 ** -11) * want.abs() + (2.0 ** -25 if dtype == HF else 0)).all(), e
    assert ops.status() == 0


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_beside_ordinary_rows(d, dtype):
    """Loud and ordinary rows by turns, in the same blocks."""
    lens, counts = [70, 300, 1900], [30, 141, 50]
    pages, scales, table, q, best = loud(lens, counts, 4, 2, 16, d, 1)
    q = q * 2.0 ** 30
    q[:, :, ::2] = queries(4, sum(counts), d, F)[:, :, ::2] * d ** -0.5
    q = q.to(dtype)
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), 1.0)
    want = values(pages, scales, table, lens, counts, 2, best)[:, 1::2]
    assert ((got[0, :, 1::2].double() - want).abs() <= (ref.UNIT[dtype] + 2.0 ** -11) * want.abs()).all()
    o, a = expect(q, pages, scales, table, lens, counts, 1.0)
    close(got[:, :, ::2], o[:, ::2], a[:, ::2], dtype)
    assert ops.status() == 0
