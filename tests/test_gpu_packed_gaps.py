"""Packed prompts whose bounds leave rows out: rows before the first prompt and behind the last belong to none and give
zeros."""
import pytest
import torch

from larder_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cu,T", [([20, 100, 300], 300), ([20, 100, 300], 350), ([1, 1, 1], 1), ([300, 300], 300),
                                  ([700, 800, 4200], 4300), ([700, 4200], 4300)], ids=str)
def test_rows_before_the_first_prompt(cu, T, D, dtype):
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(1, T, h, D, generator=g).to(dtype).cuda().transpose(1, 2) for h in (4, 2, 2))
    out = torch.full_like(q, 9.0)
    ops.attn_packed(q, k, v, 0.1, torch.tensor(cu, dtype=torch.int32).cuda(), out=out)
    a, b = cu[0], cu[-1]
    assert (out[:, :, :a] == 0).all() and (out[:, :, b:] == 0).all()
    if b > a:  # the prompts themselves: as without the rows around them
        inner = torch.tensor([c - a for c in cu], dtype=torch.int32).cuda()
        o = ops.attn_packed(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], 0.1, inner)
        u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 1e-4}[dtype]
        assert (out[:, :, a:b].double() - o.double()).abs().max() <= 6 * u * v.abs().max()
    assert ops.status() == 0
