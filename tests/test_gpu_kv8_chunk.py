"""Attention of packed chunks of new tokens over the paged 8-bit cache, against 64 bits.

Codes are exact in f16 and in fp32, queries go to f16 exactly (bf16 rows shifted by a power of two), scores are fp32 sums of D
products, weights are rounded to f16 (2^-11 of each) before the second product, whose sums are fp32; the result is rounded
once (u). Scores of these sizes (|s| < 32 in base 2) are off by less than 2^-13 (D roundings of 2^-24 relative to partial sums
below 64, the factor's), so a weight is off by 2^-11 + 2^-13, the sum of weights too, and |err| <= u |o| + 2^-9 sum p |v|.
fp32: 1e-4 sum p |v|."""
import math

import pytest
import torch

from larder_b200 import kv8, ops
from larder_b200.rope import Rope

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def cache(lens, hk, page, d, seed=0, spread=0.0, num=None):
    """Pages in no order with codes of random values for sequences of these lengths; all else is arbitrary bytes (NaN codes
    among them), NaN scales and table entries out of any range."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = [-(-n // page) for n in lens]
    num = num or sum(per) + 2
    pages = torch.randint(0, 256, (num, 2, hk, page, d), generator=g, dtype=torch.uint8, device="cuda")
    scales = torch.full((num, 2, hk), float("nan"), device="cuda")
    ids = torch.randperm(num, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(per + [1])), 1 << 30, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(per[b]):
            i = ids.pop()
            table[b, j] = i
            rows = min(page, n - j * page)
            x = torch.randn(2, hk, rows, d, generator=g, device="cuda")
            s = torch.exp2(torch.randint(-9, -7, (2, hk), generator=g, device="cuda").float())
            if spread:
                s *= torch.exp2((spread * torch.randn(2, hk, generator=g, device="cuda")).round())
            pages[i, :, :, :rows] = (x * 64).to(torch.float8_e4m3fn).view(torch.uint8)
            scales[i] = s
    return pages.view(torch.float8_e4m3fn), scales, table.cuda()


def expect(q, pages, scales, table, lens, counts, scale, causal=True, first=0):
    """(o, sum p |v|) fp64 [Hq, T, D] for q [1, Hq, T, D]: sequence b's rows follow one another from `first`."""
    _, Hq, T, D = q.shape
    Hk = pages.shape[2]
    o = torch.zeros(Hq, T, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    at = first
    for b, (L, n) in enumerate(zip(lens, counts)):
        if n == 0:
            continue
        seen = (L - n + 1 + torch.arange(n, device=q.device)).clamp(0, L) if causal else torch.full((n,), L, device=q.device)
        for h in range(Hq):
            k, v = (ref.held(pages, scales, table[b], L, i, h // (Hq // Hk)) for i in (0, 1))
            s = q[0, h, at:at + n].double() @ k.T * scale
            s = s.masked_fill(torch.arange(L, device=q.device) >= seen[:, None], -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # (a row that sees nothing)
            o[h, at:at + n], a[h, at:at + n] = p @ v, p @ v.abs()
        at += n
    return o, a


def close(got, o, a, dtype):
    err = (got[0].double() - o).abs()
    tol = 1e-4 * a + 1e-30 if dtype == F else ref.UNIT[dtype] * o.abs() + 2.0 ** -9 * a + 1e-7
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), ((err - tol).max(), err.max())


def queries(hq, T, d, dtype, seed=0, grow=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    return (torch.randn(1, T, hq, d, generator=g, device="cuda") * grow).to(dtype).transpose(1, 2)


def run(lens, counts, hq, hk, page, d, dtype, causal=True, seed=0, scale=None, spread=0.0, q=None):
    pages, scales, table = cache(lens, hk, page, d, seed, spread)
    q = queries(hq, sum(counts), d, dtype, seed) if q is None else q
    scale = d ** -0.5 if scale is None else scale
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), scale, causal)
    assert ops.status() == 0 and got.shape == q.shape and got.dtype is q.dtype
    close(got, *expect(q, pages, scales, table, lens, counts, scale, causal), dtype)
    return got


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("hq,hk", [(4, 1), (6, 2), (7, 1), (3, 3), (40, 2)])
@pytest.mark.parametrize("page,d", [(16, 64), (64, 128), (32, 256), (128, 128)])
def test_ragged_chunks(page, d, hq, hk, dtype):
    """New tokens from none to a few tiles' worth, behind nothing or behind a prefix that ends inside pages and tiles."""
    run([1, 40, 300, 129, 70, 5], [1, 33, 0, 129, 64, 5], hq, hk, page, d, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_prefixes(d, dtype):
    """Few rows over many tiles (the keys are split over the CTAs), and many rows over many tiles."""
    run([5000, 77], [3, 2], 8, 2, 64, d, dtype)
    run([3001], [700], 4, 2, 16, d, dtype)
    run([9000], [1], 1, 1, 32, d, dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, F])
def test_not_causal(d, dtype):
    run([200, 513, 0, 31], [40, 1, 3, 31], 4, 2, 32, d, dtype, causal=False)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_more_new_tokens_than_cached(dtype):
    """Rows before the first cached token see nothing and give zeros; a sequence without any."""
    got = run([5, 0, 130], [20, 7, 131], 4, 2, 16, 128, dtype)
    assert (got[:, :, :15] == 0).all() and (got[:, :, 20:27] == 0).all() and (got[:, :, 27] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("d", [64, 256])
def test_rows_of_no_sequence(d, dtype):
    """Rows before cu[0] and from cu[B] on give zeros, whatever the output held."""
    pages, scales, table = cache([50, 300], 2, 16, d)
    q = queries(4, 900, d, dtype)
    out = torch.full_like(q, float("nan"))
    ops.kv8_attend_packed(q, pages, scales, table, i32([50, 300]), i32([300, 310, 420]), d ** -0.5, out=out)
    assert ops.status() == 0
    assert (out[:, :, :300] == 0).all() and (out[:, :, 420:] == 0).all()
    close(out[:, :, 300:420], *(t[:, 300:420] for t in expect(q, pages, scales, table, [50, 300], [10, 110], d ** -0.5, first=300)),
          dtype)
    ops.kv8_attend_packed(q, pages, scales, table, i32([50, 300]), i32([900, 900, 900]), d ** -0.5, out=out)
    assert (out == 0).all() and ops.status() == 0


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_strides_and_alignment(d, dtype):
    """Queries and outputs as slices of wider rows, off the 16-byte grid, heads-first and token-first."""
    lens, counts = [90, 400], [30, 141]
    pages, scales, table = cache(lens, 2, 32, d)
    T = sum(counts)
    base = queries(6, T, d, dtype)
    want = expect(base, pages, scales, table, lens, counts, 0.1)
    for off, pad in ((0, 0), (1, 3), (8, 16), (4, 4)):
        wide = torch.zeros(T, 6, d + off + pad, dtype=dtype, device="cuda")
        q = wide[:, :, off:off + d].transpose(0, 1)[None]
        q.copy_(base)
        room = torch.full((6, T, d + off + pad), 7.0, dtype=dtype, device="cuda")
        out = room[:, :, off:off + d][None]
        ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), 0.1, out=out)
        close(out, *want, dtype)
        assert (room[:, :, :off] == 7).all() and (room[:, :, off + d:] == 7).all()
    close(ops.kv8_attend_packed(base.contiguous(), pages, scales, table, i32(lens), i32(starts(counts)), 0.1), *want, dtype)
    one = base[:, :1, :1].expand(1, 6, T, d)  # rows that overlap in memory
    close(ops.kv8_attend_packed(one, pages, scales, table, i32(lens), i32(starts(counts)), 0.1),
          *expect(one, pages, scales, table, lens, counts, 0.1), dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_scales_far_apart(d, dtype):
    """Pages whose scales differ by powers of two up to 2^20 and more: the weights carry the values' scale."""
    run([700], [200], 4, 2, 16, d, dtype, spread=2.0)
    pages, scales, table = cache([300], 1, 16, d)
    q = queries(4, 60, d, dtype)
    ids = table[0, :19].long()
    scales[ids, 1] *= torch.exp2(torch.arange(19, device="cuda").float() * 12 - 130)[:, None]  # some below 2^-100
    scales[ids[3]], pages.view(torch.uint8)[ids[3]] = 0.0, 0  # a page of zeros
    scales[ids[5], 0], pages.view(torch.uint8)[ids[5], 0] = 0.0, 0
    got = ops.kv8_attend_packed(q, pages, scales, table, i32([300]), i32([0, 60]), d ** -0.5)
    o, a = expect(q, pages, scales, table, [300], [60], d ** -0.5)
    if dtype is HF:  # values reach 2^80: past f16's range the result is an infinity
        over = o.abs() - 2.0 ** -9 * a >= 65520
        assert over.any() and torch.equal(got[0][over].double(), torch.sign(o[over]) * math.inf)
        unsure = o.abs() + 2.0 ** -9 * a >= 65504
        got, o, a = got.masked_fill(unsure, 0), o.masked_fill(unsure, 0), a.masked_fill(unsure, 0)
    close(got, o, a, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_key_that_dominates_with_a_value_of_zero(d, dtype):
    """The first key takes nearly all the weight and its value is zero: the others keep their precision."""
    L, n = 400, 150
    pages, scales, table = cache([L], 1, 16, d)
    q = queries(2, n, d, dtype).abs() + 0.5
    raw, i = pages.view(torch.uint8), int(table[0, 0])
    raw[i, 0, 0, 0] = torch.full((d,), 30.0, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    scales[i, 0, 0] = 2.0 ** -5
    raw[i, 1, 0, 0] = 0
    scale = 12.0 / (30 * 2.0 ** -5 * d * 1.3)  # the sink's score is about 12: weights e^-12 for the others
    got = ops.kv8_attend_packed(q, pages, scales, table, i32([L]), i32([0, n]), scale)
    close(got, *(t for t in expect(q, pages, scales, table, [L], [n], scale)), dtype)
    o, a = expect(q, pages, scales, table, [L], [n], scale)
    assert ((got[0].double() - o).abs() <= ref.UNIT[dtype] * o.abs() + 2.0 ** -9 * a + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_codes_reach_the_rows_that_see_them_only(d, dtype):
    """A NaN value or key of a new token: rows before it are as without it; rows that see a NaN key are NaN, a NaN value in
    its column only."""
    lens, counts, hq = [300, 260], [140, 100], 2
    pages, scales, table = cache(lens, 1, 16, d)
    q = queries(hq, sum(counts), d, dtype)
    want, a = expect(q, pages, scales, table, lens, counts, 0.1)
    raw = pages.view(torch.uint8)

    def put(b, pos, kind, dim):
        raw[int(table[b, pos // 16]), kind, 0, pos % 16, dim] = 0x7F

    put(0, 200, 1, 5)   # sequence 0, its new token 40: a value
    put(1, 230, 0, 9)   # sequence 1, its new token 70: a key
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(starts(counts)), 0.1)
    assert ops.status() == 0
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, :, 40:140, 5] = True
    bad[:, :, 140 + 70:] = True
    assert torch.equal(torch.isnan(got), bad)
    fine = torch.where(bad, torch.zeros_like(got), got)
    close(fine, want.masked_fill(bad[0], 0), a, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_infinite_and_nan_queries(d, dtype):
    """A query that is not finite spoils its own row."""
    lens, counts = [500], [130]
    pages, scales, table = cache(lens, 2, 32, d)
    q = queries(4, 130, d, dtype).contiguous()
    want, a = expect(q, pages, scales, table, lens, counts, 0.1)
    q[0, 1, 7, 3] = float("nan")
    q[0, 2, 100, 0] = float("inf")
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32([0, 130]), 0.1)
    assert torch.isnan(got[0, 1, 7]).all() and torch.isnan(got[0, 2, 100]).all()
    for h, t in ((1, 7), (2, 100)):
        got[0, h, t], want[h, t], a[h, t] = 0, 0, 0
    close(got, want, a, dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_sizes_of_queries_and_scale(dtype):
    """Small and large queries (bf16 rows are shifted into f16's range), a negative scale, a scale of zero."""
    lens, counts = [200], [40]
    pages, scales, table = cache(lens, 2, 16, 128)
    base = queries(4, 40, 128, F)
    for grow, scale in ((1.0, -0.09), (1.0, 0.0), (2.0 ** 12, 0.09 * 2.0 ** -12), (2.0 ** -12, 0.09 * 2.0 ** 12)):
        q = (base * grow).to(dtype)
        if dtype is HF and grow < 1:
            q = (base.round() * grow).to(dtype)  # (exact in f16's subnormals)
        got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32([0, 40]), scale)
        close(got, *expect(q, pages, scales, table, lens, counts, scale), dtype)
    if dtype is BF:
        q = (base * 1e30).to(BF)
        got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32([0, 40]), 0.09e-30)
        close(got, *expect(q, pages, scales, table, lens, counts, 0.09e-30), BF)


@pytest.mark.parametrize("B", [1500])
def test_many_sequences(B):
    """More sequences than one launch takes, empty ones among them, rows of no sequence at both ends."""
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 3, (B,), generator=g).tolist()
    lens = [c + int(x) for c, x in zip(counts, torch.randint(0, 40, (B,), generator=g))]
    pages, scales, table = cache(lens, 1, 16, 64)
    T = sum(counts)
    q = queries(2, T + 9, 64, BF)
    cu = [x + 4 for x in starts(counts)]
    got = ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(cu), 0.125)
    assert ops.status() == 0
    o, a = expect(q, pages, scales, table, lens, counts, 0.125, first=4)
    close(got, o, a, BF)
    assert (got[:, :, :4] == 0).all() and (got[:, :, 4 + T:] == 0).all()


def test_agrees_with_the_cut_into_smaller_chunks():
    """A prompt in one chunk, in chunks of uneven lengths, and a token at a time (kv8_attend) give the same attention."""
    c = kv8.Cache(64, 16, 2, 128)
    rope = Rope(128)
    T = 400
    k, v = (queries(2, T, 128, BF, seed=s) for s in (1, 2))
    q = queries(8, T, 128, BF)
    outs = []
    for cuts in ([T], [1, 150, 49, 200]):
        h, at, o = c.add(), 0, []
        for n in cuts:
            step = c.step([h], [n])
            c.append(step, k[:, :, at:at + n], v[:, :, at:at + n], rope=rope, packed=True)
            o.append(c.attend(step, rope.apply(q[:, :, at:at + n], step.positions), 0.1, packed=True))
            at += n
        outs.append(torch.cat(o, 2))
        last = c.step([h], [0])
        one = ops.kv8_attend(rope.apply(q[:, :, -1:], i32([[T - 1]])), c.pages, c.scales, last.table, last.kv_len, 0.1)
        assert ((one - outs[-1][:, :, -1:]).abs().float() <= 2.0 ** -7 * one.abs().float() + 2e-3).all()
        c.drop(h)
    assert ((outs[0] - outs[1]).abs().float() <= 2.0 ** -7 * outs[0].abs().float() + 4e-3).all()


def test_the_same_bits_again_and_in_a_graph_and_on_another_stream():
    lens, counts, args = [3000, 900, 40], [50, 300, 40], {}
    for d, dtype in ((128, BF), (256, HF), (64, HF)):
        pages, scales, table = cache(lens, 2, 32, d)
        q = queries(8, sum(counts), d, dtype)
        args = (q, pages, scales, table, i32(lens), i32(starts(counts)), 0.1)
        first = ops.kv8_attend_packed(*args)
        for _ in range(3):
            assert torch.equal(first, ops.kv8_attend_packed(*args))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a = ops.kv8_attend_packed(*args)
            b = ops.kv8_attend_packed(*args)
        for _ in range(2):
            a.zero_(), b.zero_()
            g.replay()
            assert torch.equal(first, a) and torch.equal(first, b)
        side = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        outs = []
        for s in side * 2:
            with torch.cuda.stream(s):
                outs.append(ops.kv8_attend_packed(*args))
        torch.cuda.synchronize()
        assert all(torch.equal(first, o) for o in outs) and ops.status() == 0


def test_lengths_change_between_replays():
    """A captured call reads its lengths, bounds and table when it runs."""
    pages, scales, table = cache([600, 600], 2, 16, 128)
    q = queries(4, 64, 128, BF)
    kv_len, cu = i32([600, 600]), i32([0, 32, 64])
    g = torch.cuda.CUDAGraph()
    ops.kv8_attend_packed(q, pages, scales, table, kv_len, cu, 0.1)
    with torch.cuda.graph(g):
        out = ops.kv8_attend_packed(q, pages, scales, table, kv_len, cu, 0.1)
    for lens, counts in (([600, 600], [32, 32]), ([64, 5], [60, 4]), ([33, 590], [0, 64]), ([1, 0], [1, 2])):
        kv_len.copy_(i32(lens))
        cu.copy_(i32(starts(counts)))
        g.replay()
        close(out, *expect(q, pages, scales, table, lens, counts, 0.1), BF)
        assert (out[:, :, sum(counts):] == 0).all()


def test_offsets_past_32_bits():
    """Page ids whose codes lie past 2^32 bytes of the pool."""
    num = (1 << 32) // (2 * 8 * 128 * 128) + 40
    pages = torch.zeros(num, 2, 8, 128, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros(num, 2, 8, device="cuda")
    p, s, t = cache([700], 8, 128, 128)
    hi = num - 1 - t
    raw = pages.view(torch.uint8)
    for j in range(6):
        raw[int(hi[0, j])], scales[int(hi[0, j])] = p.view(torch.uint8)[int(t[0, j])], s[int(t[0, j])]
    q = queries(16, 90, 128, BF)
    want = ops.kv8_attend_packed(q, p, s, t, i32([700]), i32([0, 90]), 0.1)
    got = ops.kv8_attend_packed(q, pages, scales, hi, i32([700]), i32([0, 90]), 0.1)
    assert torch.equal(want, got) and ops.status() == 0


def test_bad_lengths_bounds_and_pages():
    """Reported through the status, read nowhere; other sequences' rows are as they should be."""
    lens, counts = [100, 90], [20, 30]
    for d in (64, 128, 256):
        for dtype in (BF, F):
            pages, scales, table = cache(lens, 2, 16, d)
            q = queries(4, 50, d, dtype)
            want, a = expect(q, pages, scales, table, lens, counts, 0.1)
            for bad in (-1, pages.shape[0], 1 << 30):
                t = table.clone()
                t[0, 2] = bad
                got = ops.kv8_attend_packed(q, pages, scales, t, i32(lens), i32([0, 20, 50]), 0.1)
                assert ops.status() != 0 and ops.status() == 0
                close(got[:, :, 20:], want[:, 20:], a[:, 20:], dtype)
            got = ops.kv8_attend_packed(q, pages, scales, table[:, :6], i32([100, -3]), i32([0, 20, 50]), 0.1)
            assert ops.status() != 0 and (got[:, :, 20:] == 0).all()
            ops.kv8_attend_packed(q, pages, scales, table, i32([1 << 30, 90]), i32([0, 20, 50]), 0.1)
            assert ops.status() != 0
            for cu in ([-5, 20, 50], [0, 20, 70], [0, 40, 20], [1 << 30, 20, -(1 << 30)]):
                ops.kv8_attend_packed(q, pages, scales, table, i32(lens), i32(cu), 0.1)
                assert ops.status() != 0


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_page_that_is_none_counts_as_zeros(d, dtype):
    """Its keys' scores are 0 and their weights count; a page whose scales are 0 is such a page too."""
    lens, counts = [300], [140]
    pages, scales, table = cache(lens, 2, 32, d)
    q = queries(4, 140, d, dtype)
    p, s = pages.clone(), scales.clone()
    for j in (1, 8):
        p.view(torch.uint8)[int(table[0, j])], s[int(table[0, j])] = 0, 0.0
    o, a = expect(q, p, s, table, lens, counts, 0.1)
    close(ops.kv8_attend_packed(q, p, s, table, i32(lens), i32([0, 140]), 0.1), o, a, dtype)
    assert ops.status() == 0
    t = table.clone()
    t[0, 1], t[0, 8] = -7, pages.shape[0]
    close(ops.kv8_attend_packed(q, pages, scales, t, i32(lens), i32([0, 140]), 0.1), o, a, dtype)
    assert ops.status() != 0


def test_beside_the_other_kernels_of_the_cache():
    """Calls of several kernels that hold tensor memory, on several streams at once."""
    lens, counts = [900, 333, 64], [200, 33, 64]
    streams = [torch.cuda.Stream() for _ in range(4)]
    work = []
    for d, dtype in ((64, BF), (128, HF), (256, BF)):
        pages, scales, table = cache(lens, 2, 32, d)
        q = queries(8, 297, d, dtype)
        k = queries(2, 297, d, dtype, seed=3)
        args = (q, pages, scales, table, i32(lens), i32(starts(counts)), 0.1)
        cu = args[5]
        work.append((lambda args=args: ops.kv8_attend_packed(*args)))
        work.append((lambda q=q, k=k, cu=cu: ops.attn_packed(q, k, k, 0.1, cu)))
    first = [w() for w in work]
    torch.cuda.synchronize()
    outs = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 4]):
            outs.append((i % len(work), work[i % len(work)]()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first[i]) for i, o in outs) and ops.status() == 0


def test_refusals():
    pages, scales, table = cache([100], 2, 16, 128)
    q, n, cu = queries(4, 10, 128, BF), i32([100]), i32([0, 10])

    def call(**kw):
        a = {"q": q, "pages": pages, "scales": scales, "table": table, "kv_len": n, "cu": cu, "scale": 0.1, **kw}
        return ops.kv8_attend_packed(**a)

    call()
    for bad in ({"q": q[0]}, {"q": q[..., :64]}, {"q": q.expand(2, 4, 10, 128)}, {"q": queries(3, 10, 128, BF)},
                {"q": q.transpose(2, 3).contiguous().transpose(2, 3)}, {"q": q.double()}, {"q": q.cpu()},
                {"kv_len": n.long()}, {"kv_len": n.cpu()}, {"kv_len": i32([1, 2])}, {"cu": i32([0])}, {"cu": cu.float()},
                {"scale": float("nan")}, {"scale": float("inf")}, {"out": torch.empty_like(q[:, :2])},
                {"out": torch.empty_like(q, dtype=HF)}, {"pages": pages[..., :96]}, {"scales": scales[1:]},
                {"table": table.long()}, {"table": table[0]}):
        with pytest.raises(ValueError):
            call(**bad)
    assert ops.kv8_attend_packed(q[:, :, :0], pages, scales, table, n, i32([0, 0]), 0.1).shape == (1, 4, 0, 128)
    assert ops.status() == 0
