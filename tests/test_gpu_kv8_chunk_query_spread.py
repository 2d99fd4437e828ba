"""bf16 queries with one dim far above the others, whose K codes are zero, so that the small ones carry the score.

A row is held in f16, its largest value at [2^14, 2^15). f16's steps end at 2^-24: a bf16 value (8 bits) of 2^-31 of the row's
largest has its last bit at or above 2^-38 of it, 2^-24 or more as it is held, and is exact; any smaller one is off by half a step
at most, 2^-25, which is 2^-39 of the largest. Scores are then off by e = scale 2^-39 max|q| max_k sum|k|, weights by factors up
to exp(2 e), results by (exp(2 e) - 1) sum p |v| beyond test_gpu_kv8_chunk's bound."""
import math

import pytest
import torch

from larder_b200 import ops

import serve_ref as ref
from test_gpu_kv8_chunk import BF, F, cache, close, expect, i32, queries, starts

pytestmark = pytest.mark.gpu


def case(d, power, dtype=BF):
    lens, counts = [300, 900], [40, 150]
    pages, scales, table = cache(lens, 2, 32, d)
    pages.view(torch.uint8)[:, 0, :, :, 7] = 0  # the large dim's codes
    q = queries(4, sum(counts), d, F)
    q[..., 7] = (1 + torch.rand(q.shape[:3], generator=torch.Generator().manual_seed(2)).cuda()) * 2.0 ** power
    return lens, counts, pages, scales, table, q.to(dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [10, 20, 26])
def test_exact_within_the_spread(d, power):
    """Random values of 2^-4 and more (smaller ones rounded to multiples of it), up to 2^31 below the largest: as any other row."""
    lens, counts, pages, scales, table, q = case(d, power)
    small = q.abs() < 2.0 ** (power - 1)
    q = torch.where(small, (q.float() * 16).round() / 16, q.float()).to(BF)
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), d ** -0.5)
    close(got, *expect(q, pages, scales, table, lens, counts, d ** -0.5), BF)
    assert ops.status() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [32, 35, 38])
def test_bounded_past_it(d, power):
    lens, counts, pages, scales, table, q = case(d, power)
    scale = d ** -0.5
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), scale)
    o, a = expect(q, pages, scales, table, lens, counts, scale)
    err, at = (got[0].double() - o).abs(), 0
    for b, n in enumerate(counts):
        for h in range(4):
            k = ref.held(pages, scales, table[b], lens[b], 0, h // 2).abs().sum(-1).max()
            e = scale * 2.0 ** -39 * q[0, h, at:at + n].double().abs().amax(-1) * k
            tol = ref.UNIT[BF] * o[h, at:at + n].abs() + (torch.exp(2 * e) - 1 + 2.0 ** -9)[:, None] * a[h, at:at + n] + 1e-7
            assert (err[h, at:at + n] <= tol).all()
            assert math.isfinite(float(e.max()))
        at += n
    assert ops.status() == 0
