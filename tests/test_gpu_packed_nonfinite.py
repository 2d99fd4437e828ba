"""Packed prompts with a NaN or an infinity among the values of a prompt of some ten thousand rows: it reaches its column in
the rows that see it, and nothing else changes: not the rows before it, which share tiles with it, nor other prompts, which
share the kernel's blocks.

Both sides of the comparison with the clean result are within u |o| + 2 u sum p |v| of the same exact one: 6 u max |v|."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
LONG = 20000


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,lens", [(64, [300, LONG, 77]), (128, [300, LONG, 77]), (256, [300, LONG, 77]),  # (256: by pairs of CTAs)
                                    (256, [300, LONG, 77] + [50] * 6)])
@pytest.mark.parametrize("at", [0, 5, 129, 9999, LONG - 1, LONG])
def test_one_value(at, D, lens, dtype):
    g = torch.Generator().manual_seed(D + len(lens))
    T, Hq, Hkv = sum(lens), 4, 2
    q, k, v = (torch.randn(1, T, h, D, generator=g).to(dtype).cuda().transpose(1, 2) for h in (Hq, Hkv, Hkv))
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()
    clean = ops.attn_packed(q, k, v, D ** -0.5, cu)
    row = 300 + at  # (LONG: the first of the prompt behind)
    end = 300 + LONG if at < LONG else 377 + LONG
    for x in (float("nan"), float("-inf")):
        v[0, 1, row, 3] = x
        o = ops.attn_packed(q, k, v, D ** -0.5, cu)
        bad = torch.zeros_like(o, dtype=torch.bool)
        bad[0, 2:, row:end, 3] = True
        assert torch.equal(~torch.isfinite(o), bad)
        assert (o - clean)[~bad].abs().max() <= 6 * ref.UNIT[dtype] * v[torch.isfinite(v)].abs().max()
    assert ops.status() == 0


@pytest.mark.parametrize("D,lens", [(64, [700, 500]), (128, [700, 500]), (256, [700, 500]), (256, [3500])])
def test_many_values(D, lens):
    """Infinities at a prompt's start, which every row sees, and NaN strewn through it: each row is right column by column."""
    g = torch.Generator().manual_seed(D)
    T = sum(lens)
    q, k, v = (torch.randn(1, T, 2, D, generator=g).to(BF).cuda().transpose(1, 2) for _ in range(3))
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()
    clean = ops.attn_packed(q, k, v, D ** -0.5, cu)
    v[0, 0, 2, 0] = v[0, 1, lens[0] - 1, D - 1] = float("inf")
    v[0, :, 1::31, 7::19] = float("nan")
    o = ops.attn_packed(q, k, v, D ** -0.5, cu)
    at = 0
    for n in lens:
        seen = torch.cummax((~torch.isfinite(v[0, :, at:at + n])).int(), 1).values.bool()
        got = o[0, :, at:at + n]
        assert torch.equal(~torch.isfinite(got), seen)
        assert (got - clean[0, :, at:at + n])[~seen].abs().max() <= 6 * 2.0 ** -8 * v[torch.isfinite(v)].abs().max()
        at += n
    assert ops.status() == 0
