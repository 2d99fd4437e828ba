"""Rotary positions on the GPU against the formula in 64 bits.

Tolerance: the angle's fraction of a turn is exact to position * 2^-65, its fp32 form and sincospi are within 2^-21 in
value, the two products and the sum add 3 * 2^-24 of |x0| + |x1|; together under 2^-20 amp (|x0| + |x1|). The result is
rounded once to the type: one unit of relative rounding more (and 2^-25 for f16's subnormals)."""
import pytest
import torch

from larder_b200 import ops
from larder_b200.rope import Rope

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def check(y, x, pos, r, inverse=False):
    want = ref.rotate(x.cpu(), pos.cpu()[:, None] if pos.dim() == 2 else pos.cpu(), r.w, r.layout, r.amp, inverse)
    tol = ref.UNIT[x.dtype] * want.abs() + 2.0 ** -20 * r.amp * ref.pair_sum(x.cpu(), r.dims, r.layout) + 2.0 ** -25
    assert y.dtype == x.dtype and y.shape == x.shape
    assert ((y.cpu().double() - want).abs() <= tol).all(), ((y.cpu().double() - want).abs() / tol).max()
    assert torch.equal(y[..., r.dims:], x[..., r.dims:])  # the dims that pass do so bit by bit


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,H,T,D,R", [(1, 1, 1, 64, 64), (16, 32, 1, 128, 128), (2, 5, 37, 128, 64), (1, 3, 301, 256, 64),
                                       (3, 2, 7, 64, 16), (1, 2, 5, 80, 48), (2, 3, 9, 66, 22), (1, 1, 2, 2, 2),
                                       (1, 40, 4, 512, 512)])
def test_rope(dtype, layout, B, H, T, D, R):
    g = torch.Generator().manual_seed(B * 1000 + D + R)
    x = torch.randn(B, T, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32).cuda()
    r = Rope(R, layout=layout)
    check(r.apply(x, pos), x, pos, r)
    check(r.apply(x, pos, inverse=True), x, pos, r, True)


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": 8.0}, {"kind": "ntk", "factor": 4.0},
                                     {"kind": "yarn", "factor": 16.0, "original": 8192}])
def test_scaled_far_positions(scaling):
    x = torch.randn(1, 4, 6, 128, generator=torch.Generator().manual_seed(3)).cuda()
    pos = torch.tensor([0, 1, 131071, 1 << 24, (1 << 31) - 2, (1 << 31) - 1], dtype=torch.int32).cuda()
    r = Rope(128, base=500000.0, scaling=scaling)
    check(r.apply(x, pos), x, pos, r)


def test_strides_offsets_and_in_place():
    g = torch.Generator().manual_seed(5)
    r = Rope(64)
    big = torch.randn(2, 11, 3 * 128 + 2, generator=g).to(BF).cuda()
    pos = torch.arange(11, dtype=torch.int32).cuda()
    for at in (0, 1, 8):  # a slice of a wider row: odd strides and offsets that 16-byte accesses do not fit
        x = big[..., at:at + 3 * 128 - 8].unflatten(-1, (4, 94))[..., :94].transpose(1, 2)
        check(r.apply(x, pos), x, pos, r)
    x = torch.randn(2, 3, 11, 128, generator=g).to(HF).cuda()
    want = r.apply(x, pos)
    y = x.clone()
    assert r.apply(y, pos, out=y) is y and torch.equal(y, want)
    z = torch.full((2, 3, 11, 256), 7.0, dtype=HF, device="cuda")
    r.apply(x, pos, out=z[..., 64:192])
    assert torch.equal(z[..., 64:192], want) and (z[..., :64] == 7).all() and (z[..., 192:] == 7).all()


def test_inverse_is_the_gradient():
    """<dy, rope(x + d)> - <dy, rope(x)> against <rope_inverse(dy), d>: the map is linear, so differences are exact up to
    rounding; and the inverse undoes the map when amp is 1."""
    g = torch.Generator().manual_seed(7)
    for layout in ("half", "interleaved"):
        for scaling in (None, {"kind": "yarn", "factor": 4.0, "original": 4096}):
            r = Rope(96, layout=layout, scaling=scaling)
            x, d, dy = (torch.randn(1, 2, 33, 128, generator=g).cuda() for _ in range(3))
            pos = torch.randint(0, 100000, (33,), generator=g, dtype=torch.int32).cuda()
            diff = ((r.apply(x + d, pos).double() - r.apply(x, pos).double()) * dy.double()).sum()
            dot = (r.apply(dy, pos, inverse=True).double() * d.double()).sum()
            # each of the 8448 products carries at most about 8 * 2^-20 amp of absolute error
            assert abs(diff - dot) <= 8448 * 8 * 2.0 ** -20 * r.amp
            if scaling is None:
                back = r.apply(r.apply(x, pos), pos, inverse=True)
                assert (back - x).abs().max() <= 2.0 ** -18 * 2 * x.abs().max()


def test_special_values_stay_in_their_pair_and_row():
    r = Rope(8)
    x = torch.ones(1, 1, 3, 16).cuda()
    x[0, 0, 1, 0] = float("nan")
    x[0, 0, 1, 15] = float("inf")
    pos = torch.arange(3, dtype=torch.int32).cuda()
    y = r.apply(x, pos)
    bad = ~torch.isfinite(y[0, 0])
    assert bad.nonzero().tolist() == [[1, 0], [1, 4], [1, 15]]


def test_another_stream():
    r = Rope(128)
    x = torch.randn(1, 8, 500, 128, device="cuda")
    pos = torch.arange(500, dtype=torch.int32, device="cuda")
    want = r.apply(x, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = r.apply(x, pos)
    s.synchronize()
    assert torch.equal(y, want) and ops.status() == 0


def test_empty_and_refused():
    r = Rope(64)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert r.apply(torch.zeros(0, 2, 4, 128, device="cuda"), pos).shape == (0, 2, 4, 128)
    x = torch.zeros(1, 2, 4, 128, device="cuda")
    for bad in (lambda: r.apply(x[..., :32], pos), lambda: r.apply(x, pos.long()), lambda: r.apply(x, pos[:3]),
                lambda: r.apply(x.transpose(-1, -2), pos), lambda: r.apply(x.double(), pos),
                lambda: r.apply(x, pos, out=x[:, :1]), lambda: r.apply(x[0], pos),
                lambda: ops.rope(x, pos, r.turns.float()), lambda: ops.rope(x, pos, r.turns, "pairs"),
                lambda: r.apply(torch.zeros(1, 1, 4, 127, device="cuda"), pos), lambda: r.apply(x.cpu(), pos)):
        with pytest.raises(ValueError):
            bad()
