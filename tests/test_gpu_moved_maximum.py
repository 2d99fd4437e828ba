"""Prefill attention where one row alone of its tile finds a far larger score late: what it has accumulated has to be scaled
down in every column, also by the warps whose own share of the keys had weights of 0 so far.

Row `row`'s scores are 200 at key `first`, 400 at key `second` and 0 elsewhere; every other row's are 0, so that no
neighbour causes the scaling. Tolerance: weights and outputs in 16 bits: u |o| + 2 u sum p |v|."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu
KEYS = [(5, 300), (40, 300), (70, 300), (100, 300), (5, 64), (130, 200)]


def inputs(T, N, D, dtype, row, first, second):
    g = torch.Generator().manual_seed(first * 1000 + second)
    q, k = torch.zeros(1, 1, T, D), torch.zeros(1, 1, N, D)
    q[..., row, 0], k[..., first, 0], k[..., second, 0] = 16, 12.5, 25
    return q.to(dtype).cuda(), k.to(dtype).cuda(), torch.randn(1, 1, N, D, generator=g).to(dtype).cuda()


def check(o, q, k, v, seen):
    want, mass = ref.attend(q[0, 0], k[0, 0], v[0, 0], 1.0, seen)
    u = ref.UNIT[q.dtype]
    assert ((o[0, 0].double() - want).abs() <= u * want.abs() + 2 * u * mass).all()
    assert ops.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", [(64, 64), (64, 128), (64, 256), (200, 128), (200, 256)])
@pytest.mark.parametrize("first,second", KEYS)
def test_prefill(first, second, T, D, dtype):
    N = 400
    q, k, v = inputs(T, N, D, dtype, T - 3, first, second)
    check(ops.attn_prefill(q, k, v, 1.0), q, k, v, [N] * T)
    check(ops.attn_prefill(q, k, v, 1.0, "causal"), q, k, v, [N - T + 1 + t for t in range(T)])
    m = torch.ones(T, N, dtype=torch.bool, device="cuda")
    check(ops.attn_prefill(q, k, v, 1.0, m), q, k, v, [N] * T)
    check(ops.attn_prefill_tiled(q, k, v, 1.0, m), q, k, v, [N] * T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D", [(400, 64), (400, 128), (400, 256), (3100, 256)])
@pytest.mark.parametrize("first,second", KEYS)
def test_packed(first, second, T, D, dtype):
    for row in (second, 399):
        q, k, v = inputs(T, T, D, dtype, row, first, second)
        cu = torch.tensor([0, T], dtype=torch.int32).cuda()
        check(ops.attn_packed(q, k, v, 1.0, cu), q, k, v, [t + 1 for t in range(T)])
