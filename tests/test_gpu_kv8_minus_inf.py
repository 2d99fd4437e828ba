"""Attention over the 8-bit cache whose scores reach minus infinity."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq", [1, 12, 20])
def test_scores_of_minus_infinity(Hq, D):
    """Scores below fp32's range are -inf: weights of 0 wherever they stand, also at the row's first keys."""
    N = 300
    x = torch.zeros(5, 2, 1, 64, D)
    x.view(5, 2, 64, D)[:2, 0, :, 0] = 448  # keys 0 .. 127
    x[:, 1] = torch.randn(5, 1, 64, D, generator=torch.Generator().manual_seed(D)) * 40
    pages, scales = x.cuda().to(torch.float8_e4m3fn), torch.ones(5, 2, 1, device="cuda")
    table = torch.arange(5, dtype=torch.int32).cuda()[None]
    q = torch.zeros(1, Hq, 1, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = -3e38
    o = ops.kv8_attend(q, pages, scales, table, i32([N]), 1.0)
    v = ref.held(pages, scales, table[0], N, 1, 0)[128:]
    want, mass = v.mean(0), v.abs().mean(0)
    for h in range(Hq):
        assert ((o[0, h, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * mass).all()
