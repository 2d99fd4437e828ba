"""Rotary positions for any layout and scaling: the frequencies of a model's rotation as exact fractions of a turn.

    r = Rope(128, base=1e6, layout="half", scaling={"kind": "yarn", "factor": 4.0, "original": 32768})
    q = r.apply(q, positions)                 # [B, H, T, D], int32 positions [B, T] or [T]
    dq = r.apply(dy, positions, inverse=True) # the gradient

`dims` of each head's first values are rotated, pair i by position * w_i, w_i = base^(-2 i / dims) before scaling:
  linear  w_i / factor (positions squeezed by the factor)
  ntk     base * factor^(dims / (dims - 2)) for base: the fastest pair is kept, the slowest squeezed by the factor
  yarn    per pair between the two: pairs that turn more than beta_fast (32) times over the original length are kept,
          those that turn less than beta_slow (1) times are squeezed, a linear ramp over the pair index between; the
          rotated values are multiplied by 0.1 ln(factor) + 1

The frequencies are formed in fp64 and held as `turns`, round(2^64 w_i / 2 pi) as int64 words, which the kernels multiply
by the position in 64-bit wrap-around arithmetic.
"""
import math

import torch

from . import ops


def frequencies(dims, base=10000.0, scaling=None):
    """(w_i, i < dims / 2, in radians a position; the factor on the rotated values), as Python floats."""
    if dims < 2 or dims % 2:
        raise ValueError(f"rope: an even number of rotated dims, got {dims}")
    if not base > 1.0:
        raise ValueError(f"rope: the base must be above 1, got {base}")
    half = dims // 2
    w = [base ** (-2.0 * i / dims) for i in range(half)]
    if scaling is None:
        return w, 1.0
    kind, f = scaling.get("kind"), float(scaling.get("factor", 0.0))
    if not f >= 1.0:
        raise ValueError(f"rope: a scaling factor of at least 1, got {scaling.get('factor')}")
    known = {"linear": {"kind", "factor"}, "ntk": {"kind", "factor"},
             "yarn": {"kind", "factor", "original", "beta_fast", "beta_slow"}}
    if kind not in known:
        raise ValueError(f"rope: unknown scaling {kind!r} (linear, ntk, yarn)")
    if set(scaling) - known[kind]:
        raise ValueError(f"rope: {kind} scaling does not take {sorted(set(scaling) - known[kind])}")
    if kind == "linear":
        return [x / f for x in w], 1.0
    if kind == "ntk":
        if dims == 2:
            raise ValueError("rope: ntk scaling needs more than one pair")
        b = base * f ** (dims / (dims - 2))
        return [b ** (-2.0 * i / dims) for i in range(half)], 1.0
    n = float(scaling.get("original", 0))
    if not n > 0:
        raise ValueError("rope: yarn scaling needs the original length")

    def pair_of(turns):  # the pair index whose angle makes so many turns over the original length
        return dims * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo = max(math.floor(pair_of(float(scaling.get("beta_fast", 32.0)))), 0)
    hi = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1.0)))), dims - 1)
    hi = hi if hi > lo else lo + 0.001
    ramp = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(half)]
    return [x + (x / f - x) * r for x, r in zip(w, ramp)], 0.1 * math.log(f) + 1.0


def turns_of(w, device=None):
    """Angles a position (radians) as int64 words of 2^-64 turns."""
    t = [int(round(x / (2 * math.pi) * 2.0 ** 64)) & (1 << 64) - 1 for x in w]
    return torch.tensor([x - (1 << 64) if x >> 63 else x for x in t], dtype=torch.int64, device=device)


class Rope:
    def __init__(self, dims, base=10000.0, layout="half", scaling=None, device="cuda"):
        ops._interleaved(layout, "Rope")
        self.dims, self.layout = dims, layout
        self.w, self.amp = frequencies(dims, base, scaling)
        self.turns = turns_of(self.w, device)

    def apply(self, x, positions, inverse=False, out=None):
        """x [B, H, T, D] rotated by positions int32 [B, T] or [T], in autograd's graph where x requires a gradient;
        inverse=True is the gradient by hand."""
        return ops.rope(x, positions, self.turns, self.layout, self.amp, inverse, out)


__all__ = ["Rope", "frequencies", "turns_of"]
