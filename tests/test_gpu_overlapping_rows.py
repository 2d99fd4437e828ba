"""Queries whose rows overlap in memory: the result is laid out as usual."""
import pytest
import torch

from larder_b200 import ops

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_overlapping_query_rows(dtype):
    """Queries whose T axis steps by one element (windows of one row): the result is laid out as usual."""
    D, N = 64, 50
    pages = (torch.randn(4, 2, 1, 16, D, generator=torch.Generator().manual_seed(1)) * 40).cuda().to(torch.float8_e4m3fn)
    scales, table = torch.full((4, 2, 1), 0.02, device="cuda"), i32([[2, 0, 3, 1]])
    flat = torch.randn(1, 4, D + 8, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    q = flat.as_strided((1, 4, 8, D), (4 * (D + 8), D + 8, 1, 1))
    o = ops.kv8_attend(q, pages, scales, table, i32([N]), 0.1)
    assert o.stride(-1) == 1
    assert torch.equal(o, ops.kv8_attend(q.contiguous(), pages, scales, table, i32([N]), 0.1))
    kk, vv = (torch.randn(1, 4, 8, D, generator=torch.Generator().manual_seed(i)).cuda() for i in (3, 4))
    cu = i32([0, 3, 8])
    q32 = flat.float().as_strided((1, 4, 8, D), (4 * (D + 8), D + 8, 1, 1))
    p = ops.attn_packed(q32, kk, vv, 0.1, cu)
    assert p.stride(-1) == 1 and torch.equal(p, ops.attn_packed(q32.contiguous(), kk, vv, 0.1, cu))
    assert ops.status() == 0
