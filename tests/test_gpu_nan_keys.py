"""A NaN in a key reaches every row that sees the key, wherever the key stands in its tile, and no other row; so does an
infinite score."""
import pytest
import torch

from larder_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,T", [(64, 40), (128, 40), (128, 300), (256, 40), (256, 300)])
def test_prefill(D, T, dtype):
    g = torch.Generator().manual_seed(D + T)
    N = 320
    q, k, v = (torch.randn(1, 1, n, D, generator=g).to(dtype).cuda() for n in (T, N, N))
    for bad in (float("nan"), float("inf")):
        for key in list(range(24)) + [63, 70, 126, 127, 128, 199, 318, 319]:
            kb = k.clone()
            kb[0, 0, key, 5] = bad
            qb = q.clone()
            qb[..., 5] = 1.0  # (an infinite key: a score of +inf)
            o = ops.attn_prefill(qb, kb, v, D ** -0.5)
            assert torch.isnan(o).all(), (bad, key)
            seen = torch.arange(N - T, N, device="cuda") >= key
            o = ops.attn_prefill(qb, kb, v, D ** -0.5, "causal")
            assert torch.equal(torch.isnan(o[0, 0]), seen[:, None].expand(T, D)), (bad, key)
    assert ops.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,T", [(64, 400), (128, 400), (256, 400), (256, 3200)])
def test_packed(D, T, dtype):
    g = torch.Generator().manual_seed(D + T)
    q, k, v = (torch.randn(1, 1, T, D, generator=g).to(dtype).cuda() for _ in range(3))
    cu = torch.tensor([0, T], dtype=torch.int32).cuda()
    q[..., 5] = 1.0
    for bad in (float("nan"), float("inf")):
        for key in list(range(24)) + [63, 70, 126, 127, 128, 199, 318, T - 1]:
            kb = k.clone()
            kb[0, 0, key, 5] = bad
            o = ops.attn_packed(q, kb, v, D ** -0.5, cu)
            seen = torch.arange(T, device="cuda") >= key
            assert torch.equal(torch.isnan(o[0, 0]), seen[:, None].expand(T, D)), (bad, key)
    assert ops.status() == 0
