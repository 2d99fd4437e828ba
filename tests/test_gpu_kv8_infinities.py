"""Infinities in pages of the 8-bit cache whose finite values are all 0."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu
INF = float("inf")


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", ["wide", "any"])
def test_infinities_among_zeros(shape, dtype):
    """Where the finite values are all 0 the scale is 0; infinities are still held as the largest codes, NaN as NaN, and a
    later token that gives the page a scale finds them there, as if all had come at once."""
    D, n = 64, 9
    x = torch.zeros(2, 1, 2, n + 3, D)
    x[:, 0, 0, 2, 5], x[:, 0, 0, 4, 17], x[0, 0, 1, 8, 63] = INF, -INF, INF
    x[1, 0, 1, 3, 1] = float("nan")
    x[:, :, 0, n:] = torch.randn(2, 1, 3, D, generator=torch.Generator().manual_seed(1))
    x = x.to(dtype).cuda()
    if shape == "any":  # an odd offset: element accesses
        wide = torch.zeros(2, 1, 2, n + 3, D + 1, dtype=dtype, device="cuda")
        wide[..., 1:] = x
        x = wide[..., 1:]
    got = []
    for cuts in ([n, 3], [n + 3]):
        pages = torch.full((1, 2, 2, 16, D), 0x55, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        scales = torch.full((1, 2, 2), float("nan"), device="cuda")
        at = 0
        for m in cuts:
            ops.kv8_append(pages, scales, x[0][:, :, at:at + m], x[1][:, :, at:at + m], i32([[0]]), i32([at]))
            at += m
            if at == n:
                assert (scales == 0).all()
                c = pages[0].float()[:, :, :n]
                src = x[:, 0, :, :n].float()
                assert torch.equal(c.nan_to_num(-1), src.clamp(-448, 448).nan_to_num(-1))
        got.append((pages.float()[:, :, :, :at], scales))
    assert torch.equal(got[0][1], got[1][1])
    assert torch.equal(got[0][0].nan_to_num(-1), got[1][0].nan_to_num(-1))
    assert ops.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_infinite_values_on_a_page_of_zeros_count_as_zeros(dtype):
    """A held value is code * scale: 448 * 0 takes part as any other 0."""
    D = 128
    k = torch.randn(1, 1, 40, D, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    v = torch.zeros_like(k)
    v[0, 0, 3, 7] = INF
    v[0, 0, 20:] = 1.0
    pages = torch.zeros(3, 2, 1, 16, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales, table = torch.zeros(3, 2, 1, device="cuda"), i32([[0, 1, 2]])
    ops.kv8_append(pages, scales, k, v, table, i32([0]))
    q = torch.randn(1, 2, 1, D, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    o = ops.kv8_attend(q, pages, scales, table, i32([40]), 0.1)
    held = [ref.held(pages, scales, table[0], 40, kind, 0) for kind in (0, 1)]
    assert (held[1][3] == 0).all()
    for h in range(2):
        want, mass = ref.attend(q[0, h], *held, 0.1, [40])
        tol = ref.UNIT[dtype] * want.abs() + (1e-4 if dtype == torch.float32 else 2.0 ** -9) * mass
        assert ((o[0, h].double() - want).abs() <= tol).all()
