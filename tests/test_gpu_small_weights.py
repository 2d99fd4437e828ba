"""Attention over the cache under a key that dominates the softmax while its value is 0 (an attention sink): the result is
made of the small weights of the other keys alone, so their relative precision shows.

Every other key has the same score, 15.125 nats (21.82 bits) below the sink's. Rounded to 16-bit floats against a maximum of
1 each weight is 4.53 steps of f16's smallest, off by a tenth; against a maximum of 2^7 it is 580.1 steps, off by 2^-12.
Tolerance: the operator's own, u |o| + 2^-9 sum p |v|."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def pool(N, D, page=64):
    """One sequence of N cached tokens of one head: key 0 is 8 e_0 with value 0, the others' keys 0, values 448 x 16."""
    num = -(-N // page)
    x = torch.zeros(num, 2, 1, page, D)
    x[0, 0, 0, 0, 0] = 8
    x[:, 1] = 448
    x[0, 1, 0, 0] = 0
    scales = torch.ones(num, 2, 1)
    scales[:, 1] = 16
    return x.cuda().to(torch.float8_e4m3fn), scales.cuda(), torch.arange(num, dtype=torch.int32).cuda()[None]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,T", [(1, 1), (8, 1), (16, 1), (4, 8), (1, 4)])
@pytest.mark.parametrize("N", [40, 64, 256])
def test_cache_sink(N, Hq, T, D, dtype):
    pages, scales, table = pool(N, D)
    q = torch.zeros(1, Hq, T, D, dtype=dtype, device="cuda")
    q[..., 0] = 15.125 / 8
    o = ops.kv8_attend(q, pages, scales, table, torch.tensor([N], dtype=torch.int32).cuda(), 1.0)
    k, v = (ref.held(pages, scales, table[0], N, kind, 0) for kind in (0, 1))
    for h in range(Hq):
        want, mass = ref.attend(q[0, h], k, v, 1.0, [N - T + 1 + t for t in range(T)])
        assert ((o[0, h].double() - want).abs() <= ref.UNIT[dtype] * want.abs() + 2.0 ** -9 * mass).all()
    assert ops.status() == 0


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cache_sink_among_random_keys(D, dtype):
    """Scores within half a nat of 0, the sink at 13.5 nats: weights from 2^-20.3 of the largest on, which are normal f16
    numbers against a maximum of 2^7."""
    N, g = 500, torch.Generator().manual_seed(D)
    pages, scales, table = pool(N, D)
    x = pages.float()
    x[:, 0, 0, :, 1:] = torch.randn(x[:, 0, 0, :, 1:].shape, generator=g).cuda()
    x[0, 0, 0, 0, 1:] = 0
    x[:, 1] = torch.rand(x[:, 1].shape, generator=g).cuda() * 400 + 40
    x[0, 1, 0, 0] = 0
    pages = x.to(torch.float8_e4m3fn)
    q = torch.randn(1, 4, 1, D, generator=g) * 0.1
    q[..., 0] = 0
    s = (q[0, :, 0] @ x[:, 0, 0].reshape(-1, D)[:N].cpu().T).abs().max()
    q = (q * (0.5 / s)).to(dtype)
    q[..., 0] = 13.5 / 8
    q = q.cuda()
    o = ops.kv8_attend(q, pages, scales, table, torch.tensor([N], dtype=torch.int32).cuda(), 1.0)
    k, v = (ref.held(pages, scales, table[0], N, kind, 0) for kind in (0, 1))
    for h in range(4):
        want, mass = ref.attend(q[0, h], k, v, 1.0, [N])
        assert ((o[0, h].double() - want).abs() <= ref.UNIT[dtype] * want.abs() + 2.0 ** -9 * mass).all()
