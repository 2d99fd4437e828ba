"""Plain 64-bit forms of the paged 8-bit cache's operators, for the tests: rotary positions, the cache's codes, attention."""
import math

import torch

# largest relative rounding of a value to the type (half a unit in the last place over the least significand)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rotate(x, positions, w, layout="half", amp=1.0, inverse=False):
    """x [..., n, D] (any dtype) rotated in fp64 by positions [n] (or [..., n]) at the angles w a position."""
    x = x.double()
    R = 2 * len(w)
    a = positions.double()[..., None] * torch.tensor(w, dtype=torch.float64, device=x.device)
    c, s = torch.cos(a) * amp, torch.sin(a) * (-amp if inverse else amp)
    y = x.clone()
    if layout == "half":
        i, j = torch.arange(R // 2), torch.arange(R // 2) + R // 2
    else:
        i, j = 2 * torch.arange(R // 2), 2 * torch.arange(R // 2) + 1
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def pair_sum(x, R, layout="half"):
    """|x0| + |x1| of each rotated value's pair (|x| elsewhere), [..., D] fp64."""
    x = x.double().abs()
    y = x.clone()
    if layout == "half":
        s = x[..., :R // 2] + x[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = s, s
    else:
        s = x[..., 0:R:2] + x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = s, s
    return y


def scale_of(m):
    """The least power of two s with m <= 448 s; 0 for 0."""
    if m == 0:
        return 0.0
    s = 2.0 ** math.floor(math.log2(m / 448.0))
    while m > 448.0 * s:
        s *= 2
    return max(s, 2.0 ** -126)


def half_step(c):
    """Half the distance between e4m3 values around c (fp64 tensor, |c| <= 448)."""
    return torch.exp2(torch.floor(torch.log2(c.abs().clamp(min=2.0 ** -6))) - 4)


def held(pages, scales, table, n, kind, h):
    """Sequence row `table` [P]: its first n held values of K (0) or V (1) of one head, fp64 [n, D]."""
    page = pages.shape[3]
    ids = table[:-(-n // page)].long()
    c = pages.view(torch.uint8)[ids, kind, h].view(torch.float8_e4m3fn).double()
    return (c * scales[ids, kind, h].double()[:, None, None]).reshape(-1, pages.shape[4])[:n]


def attend(q, k, v, scale, seen):
    """Softmax attention in fp64 of q [T, D] over k, v [N, D], row t seeing keys [0, seen[t]): (o, sum_n p |v|). A key
    that a row does not see takes no part, whatever it holds."""
    o = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    for t in range(q.shape[0]):
        m = int(seen[t])
        if m > 0:
            p = torch.softmax(k[:m].double() @ q[t].double() * scale, 0)
            o[t], a[t] = p @ v[:m].double(), p @ v[:m].double().abs()
    return o, a
