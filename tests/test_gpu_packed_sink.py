"""Packed prompts under a key that dominates the softmax while its value is 0 (an attention sink): the result is made of the
small weights of the other keys alone.

Every other key has the same score, 15.125 nats (21.82 bits) below the first's. Rounded to f16 against a maximum of 1 each
weight is 4.53 steps of f16's smallest, off by a tenth; against a maximum of 2^7 it is 580.1 steps, off by 2^-12. Tolerance:
the operator's own, u |o| + 2 u sum p |v|."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,D", [(150, 64), (150, 128), (150, 256), (3100, 256)])
def test_packed_sink(T, D, dtype):
    q = torch.zeros(1, 1, T, D, dtype=dtype, device="cuda")
    k, v = torch.zeros_like(q), torch.full_like(q, 7168.0)
    q[..., 0] = 15.125 / 8
    k[:, :, 0, 0] = 8
    v[:, :, 0] = 0
    o = ops.attn_packed(q, k, v, 1.0, torch.tensor([0, T], dtype=torch.int32).cuda())
    rows = [1, 2, 63, 64, 65, 149] + ([T - 1] if T > 150 else [])
    want, mass = ref.attend(q[0, 0, rows], k[0, 0], v[0, 0], 1.0, [r + 1 for r in rows])
    u = ref.UNIT[dtype]
    assert ((o[0, 0, rows].double() - want).abs() <= u * want.abs() + 2 * u * mass).all()
    assert (o[0, 0, 0] == 0).all() and ops.status() == 0
