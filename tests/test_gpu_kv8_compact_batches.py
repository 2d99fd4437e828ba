"""Compaction of more sequences than a warp has lanes, and copies of more pages than one launch takes."""
import random

import pytest
import torch

from larder_b200 import ops
from larder_b200.rope import Rope

from test_gpu_kv8_pages import pool, run_compact, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [31, 32, 33, 64, 100, 1025])
@pytest.mark.parametrize("R", [0, 64, 10])
def test_many_sequences(B, R):
    """Empty ones, ones that keep nothing, ones of several pages, in no order."""
    rng = random.Random(B)
    page = 16
    lens = [rng.choice([0, 1, page, rng.randint(0, 5 * page)]) for _ in range(B)]
    keeps = [sorted(rng.sample(range(n), rng.choice([0, n, n // 2]))) for n in lens]
    start = [page * rng.choice([0, 0, 1, 3]) for _ in lens]
    run_compact(lens, keeps, start, 1, page, 64, Rope(R) if R else None, seed=B)


def test_copies_past_one_launch():
    n = 65535 + 1000
    pages, scales = pool(n, 1, 16, 64)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(0)).int().cuda()
    other, more = pool(n + 1, 1, 16, 64, seed=1)
    last, last_scale = other[n].clone(), more[n].clone()
    ops.kv8_copy(pages, scales, torch.arange(n, dtype=torch.int32, device="cuda"), order, into=(other, more))
    at = order.long()
    assert same(other[at], pages) and torch.equal(more[at], scales)
    assert same(other[n], last) and torch.equal(more[n], last_scale) and ops.status() == 0
