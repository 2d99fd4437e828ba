"""Gradients through the rotary positions: autograd's against the transposed rotation in 64 bits, and against differences.

The gradient is one rotation of dy: an error of 2^-18 of the pair's |dy| (the angle's and the products' fp32 roundings) and one
rounding to the type. The map is linear, so a difference quotient has the rounding of its two values alone."""
import pytest
import torch

from larder_b200 import ops
from larder_b200.rope import Rope

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def close(got, dy, pos, r, inverse):
    for b in range(got.shape[0]):
        want = ref.rotate(dy[b], pos[b] if pos.dim() == 2 else pos, r.w, r.layout, r.amp, inverse)
        tol = ref.UNIT[got.dtype] * want.abs() + 2.0 ** -18 * r.amp * ref.pair_sum(dy[b], r.dims, r.layout)
        assert ((got[b].double() - want).abs() <= tol + 1e-30).all()


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
def test_gradient(inverse, layout, dtype):
    g = torch.Generator().manual_seed(5)
    r = Rope(64, layout=layout, scaling={"kind": "yarn", "factor": 4.0, "original": 4096})
    x, dy = (torch.randn(2, 37, 3, 128, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    pos = torch.randint(0, 100000, (2, 37), generator=g, dtype=torch.int32).cuda()
    plain = r.apply(x, pos, inverse=inverse)
    x.requires_grad_()
    y = r.apply(x, pos, inverse=inverse)
    assert y.requires_grad and torch.equal(y, plain)
    y.backward(dy)
    close(x.grad, dy, pos, r, not inverse)
    assert torch.equal(x.grad, r.apply(dy, pos, inverse=not inverse))


def test_broadcast_and_strided_gradients():
    """dy as reductions and transposed consumers leave it: expanded from one value, or without a unit last stride."""
    g = torch.Generator().manual_seed(6)
    r = Rope(128)
    x = torch.randn(1, 2, 19, 128, generator=g).cuda().requires_grad_()
    pos = torch.arange(1000, 1019, dtype=torch.int32).cuda()
    r.apply(x, pos).sum().backward()
    close(x.grad, torch.ones_like(x), pos, r, True)
    x.grad = None
    w = torch.randn(1, 2, 128, 19, generator=g).cuda()
    (r.apply(x, pos).transpose(2, 3) * w).sum().backward()
    close(x.grad, w.transpose(2, 3), pos, r, True)
    base = torch.randn(1, 1, 19, 128, generator=g).cuda().requires_grad_()
    dy = torch.randn(1, 2, 19, 128, generator=g).cuda()
    r.apply(base.expand(1, 2, 19, 128), pos).backward(dy)  # heads that share their input: the sum over them
    each = sum(ref.rotate(dy[0, h], pos, r.w, inverse=True) for h in range(2))
    tol = 2.0 ** -17 * (ref.pair_sum(dy[0, 0], 128) + ref.pair_sum(dy[0, 1], 128))
    assert ((base.grad[0, 0].double() - each).abs() <= tol).all()


def test_differences_and_second_order():
    g = torch.Generator().manual_seed(7)
    r = Rope(96)
    x, d, dy = (torch.randn(1, 2, 33, 128, generator=g).cuda() for _ in range(3))
    pos = torch.randint(0, 100000, (33,), generator=g, dtype=torch.int32).cuda()
    x.requires_grad_()
    dy.requires_grad_()
    y = r.apply(x, pos)
    gx, = torch.autograd.grad(y, x, dy, create_graph=True)
    with torch.no_grad():
        diff = ((r.apply(x + d, pos).double() - r.apply(x, pos).double()) * dy.double()).sum()
    dot = (gx.double() * d.double()).sum()
    assert abs(diff - dot) <= 8448 * 8 * 2.0 ** -20  # each of the 8448 products' absolute error
    back, = torch.autograd.grad(gx, dy, d)  # the gradient is linear in dy: its gradient is the rotation itself
    close(back, d, pos, r, False)


def test_without_a_graph_and_refusals():
    r = Rope(64)
    x = torch.randn(1, 2, 5, 64).cuda().requires_grad_()
    pos = torch.arange(5, dtype=torch.int32).cuda()
    with torch.no_grad():
        y = r.apply(x, pos)
        assert not y.requires_grad and torch.equal(r.apply(x, pos, out=torch.empty_like(x)), y)
    assert torch.equal(r.apply(x.detach(), pos), y)
    with pytest.raises(ValueError, match="out"):
        r.apply(x, pos, out=torch.empty_like(x))
    with pytest.raises(ValueError):
        ops.rope(x, pos.long(), r.turns)
    z = r.apply(x, pos)
    pos.add_(1)  # what the backward pass needs has changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
