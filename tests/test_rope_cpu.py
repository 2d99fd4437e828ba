"""Rotary frequencies and their fractions of a turn (no GPU), and the refusals that need none."""
import math

import pytest
import torch

from larder_b200 import kv8, ops
from larder_b200.rope import Rope, frequencies, turns_of


def test_turns_hold_the_angle_at_any_position():
    """position * turns mod 2^64 is the angle's fraction of a turn to position * 2^-65."""
    w, _ = frequencies(128, base=500000.0)
    t = turns_of(w).tolist()
    for pos in (1, 4097, 131071, (1 << 31) - 1):
        for x, f in zip(w, t):
            got = ((pos * f) % (1 << 64)) / 2.0 ** 64 * 2 * math.pi
            want = math.fmod(pos * x, 2 * math.pi)  # fp64: off by pos * x * 2^-53
            d = abs(got - want) % (2 * math.pi)
            assert min(d, 2 * math.pi - d) <= pos * 2.0 ** -64 * 2 * math.pi + pos * x * 2.0 ** -51 + 1e-12


def test_scalings():
    w, a = frequencies(64)
    assert a == 1.0 and w[0] == 1.0 and w[31] == pytest.approx(10000.0 ** (-62 / 64))
    lin, a = frequencies(64, scaling={"kind": "linear", "factor": 4.0})
    assert a == 1.0 and lin == [x / 4.0 for x in w]
    ntk, a = frequencies(64, scaling={"kind": "ntk", "factor": 4.0})
    assert a == 1.0 and ntk[0] == w[0] and ntk[31] == pytest.approx(w[31] / 4.0)
    yarn, a = frequencies(64, scaling={"kind": "yarn", "factor": 4.0, "original": 4096})
    assert a == pytest.approx(0.1 * math.log(4.0) + 1.0)
    for x, y in zip(w, yarn):
        turns = 4096 * x / (2 * math.pi)
        if turns > 40:
            assert y == x
        if turns < 0.9:
            assert y == pytest.approx(x / 4.0)
        assert x / 4.0 - 1e-12 <= y <= x
    assert frequencies(64, scaling={"kind": "yarn", "factor": 1.0, "original": 4096}) == (w, 1.0)


@pytest.mark.parametrize("dims,base,scaling", [(0, 1e4, None), (7, 1e4, None), (64, 1.0, None),
                                               (64, 1e4, {"kind": "linear"}), (64, 1e4, {"kind": "linear", "factor": 0.5}),
                                               (64, 1e4, {"kind": "dynamic", "factor": 2.0}),
                                               (64, 1e4, {"kind": "yarn", "factor": 2.0}),
                                               (64, 1e4, {"kind": "ntk", "factor": 2.0, "original": 4096}),
                                               (2, 1e4, {"kind": "ntk", "factor": 2.0})])
def test_refused_frequencies(dims, base, scaling):
    with pytest.raises(ValueError):
        frequencies(dims, base, scaling)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        Rope(64, layout="pairs", device="cpu")
    r = Rope(64, device="cpu")
    x = torch.zeros(1, 2, 3, 64)
    pos = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        r.apply(x, pos)
    pages = torch.zeros(2, 2, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales, table = torch.zeros(2, 2, 2), torch.zeros(1, 2, dtype=torch.int32)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_append(pages, scales, x, x, table, n)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_attend(x[:, :, :1], pages, scales, table, n, 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attn_packed(x, x, x, 0.1, torch.zeros(2, dtype=torch.int32))


def test_cache_hands_out_pages():
    """The host side of the cache: tables, starts, lengths, offsets, positions; pages return when a sequence ends."""
    c = kv8.Cache(6, 16, 2, 64, device="cpu")
    a, b = c.add(), c.add()
    st = c.step([a, b], [20, 5])
    assert c.free_pages == 3 and st.table.shape == (2, 2)
    assert st.start.tolist() == [0, 0] and st.kv_len.tolist() == [20, 5] and st.cu.tolist() == [0, 20, 25]
    assert st.positions.tolist() == list(range(20)) + list(range(5))
    used = {st.table[0, 0].item(), st.table[0, 1].item(), st.table[1, 0].item()}
    assert len(used) == 3 and used <= set(range(6))
    st = c.step([b, a], [1, 1])
    assert st.start.tolist() == [5, 20] and st.positions.tolist() == [[5], [20]] and c.free_pages == 3
    with pytest.raises(ValueError, match="pages needed"):
        c.step([a], [16 * 4])
    assert c.length(a) == 21 and c.free_pages == 3
    c.trim(a, 16)
    assert c.free_pages == 4 and c.length(a) == 16
    with pytest.raises(ValueError):
        c.trim(a, 17)
    c.drop(b)
    assert c.free_pages == 5
    with pytest.raises(ValueError):
        c.step([a, a], [1, 1])
    st = c.step([a], [0])
    assert st.kv_len.tolist() == [16] and st.positions.numel() == 0
    for bad in ((0, 16, 1, 64), (4, 17, 1, 64), (4, 16, 0, 64), (4, 16, 1, 96)):
        with pytest.raises(ValueError):
            kv8.Cache(*bad, device="cpu")
