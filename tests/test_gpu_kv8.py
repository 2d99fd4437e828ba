"""The paged 8-bit KV cache on the GPU: what append leaves in the pages, and attention over them, in 64 bits.

Append. The scale is a power of two fixed by the rotated values' largest magnitude; a held value is the nearest e4m3
code: |held - x| <= half a code step, plus, for rotated keys, the error of the rotated value in fp32, whatever forms the sine
and cosine (the multi-function unit's are off by 2^-21, its argument by pi 2^-23, three fp32 roundings: under 2^-18 (|x0| +
|x1|)).
Values and held codes that are rescaled take no such error: they must be the nearest codes exactly.

Attention. Codes are exact in f16. Queries go to f16 exactly (bf16 has fewer bits, the range is shifted); scores are
fp32 sums of D products; weights are rounded to f16 (2^-11) before the second product; the result is rounded once (u).
Score errors stay under 2^-11 for these sizes, so |err| <= u |o| + 2^-9 sum p |v|. fp32: 1e-4 sum p |v|."""
import pytest
import torch

from larder_b200 import kv8, ops
from larder_b200.rope import Rope

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def pool(num, hk, page, d, seed=0):
    """Pages of arbitrary bytes (NaN codes among them) and arbitrary scales: whatever memory held before."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (num, 2, hk, page, d), generator=g, dtype=torch.uint8).cuda()
    return codes.view(torch.float8_e4m3fn), torch.full((num, 2, hk), float("nan"), device="cuda")


def tables(per, num, seed=1):
    """Shuffled pages for sequences of per[b] pages; entries past them are out of any range."""
    ids = torch.randperm(num, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(per), max(per + [1])), 1 << 30, dtype=torch.int32)
    for b, n in enumerate(per):
        for j in range(n):
            t[b, j] = ids.pop()
    return t.cuda()


def check_append(before, after, x, table, start, n, kind, rope):
    """One sequence's K (kind 0) or V rows x [hk, n, d] fp64 (unrotated) against the pools before and after."""
    (p0, s0), (p1, s1) = before, after
    page = p0.shape[3]
    y = x
    slack = torch.zeros_like(x)
    if kind == 0 and rope is not None:
        y = ref.rotate(x, torch.arange(start, start + n, device=x.device), rope.w, rope.layout, rope.amp)
        slack = 2.0 ** -18 * rope.amp * ref.pair_sum(x, rope.dims, rope.layout)
        slack[..., rope.dims:] = 0
    for j in range(start // page, (start + n - 1) // page + 1):
        lo, hi = max(start - j * page, 0), min(start + n - j * page, page)
        rows = slice(j * page + lo - start, j * page + hi - start)
        pg = int(table[j])
        for h in range(x.shape[0]):
            a, sl = y[h, rows], slack[h, rows]
            fin = torch.isfinite(a)
            was = float(s0[pg, kind, h]) if lo else 0.0
            now = max(was, ref.scale_of(float(a[fin].abs().max()) if fin.any() else 0.0))
            assert float(s1[pg, kind, h]) == now, (pg, kind, h, float(s1[pg, kind, h]), now)
            c1 = p1[pg, kind, h].double()
            if now == 0:
                assert (c1[lo:hi] == 0).all()
            else:
                z = (a / now).clamp(-448, 448)
                err = (c1[lo:hi] - z).abs()
                assert (err <= ref.half_step(z) + sl / now)[fin].all()
                assert torch.equal(torch.isnan(c1[lo:hi]), torch.isnan(a))
                inf = torch.isinf(a)
                assert torch.equal(c1[lo:hi][inf], torch.sign(a[inf]) * 448)
            old = p0[pg, kind, h, :lo].double() * (was / now if now else 0.0)
            err = (c1[:lo] - old).abs()  # rescaled codes: nearest, and no error where they stay normal
            fin = torch.isfinite(old)
            assert (err[fin] <= ref.half_step(old[fin])).all()
            assert (err[fin & ((old.abs() >= 2.0 ** -6) | (was == now))] == 0).all()
            u0, u1 = p0.view(torch.uint8), p1.view(torch.uint8)
            assert torch.equal(u0[pg, kind, h, hi:], u1[pg, kind, h, hi:])  # past the new rows: untouched


def run_append(page, d, hk, starts, counts, dtype, rope=None, packed=False, lens=False, grow=1.0, seed=0, x=None):
    g = torch.Generator().manual_seed(seed)
    B = len(starts)
    per = [-(-(s + n) // page) for s, n in zip(starts, counts)]
    num = sum(per) + 2
    pages, scales = pool(num, hk, page, d, seed)
    table = tables(per, num, seed)
    kw = {} if rope is None else {"turns": rope.turns, "layout": rope.layout, "amp": rope.amp}
    if any(starts):  # what is there already, appended as prompts
        T = max(starts)
        k, v = (torch.randn(B, T, hk, d, generator=g).cuda().transpose(1, 2) for _ in range(2))
        ops.kv8_append(pages, scales, k, v, table, i32([0] * B), lens=i32(starts), **kw)
    before = (pages.clone(), scales.clone())
    T = sum(counts) if packed else max(counts + [1])
    if x is None:
        x = [(torch.randn(1 if packed else B, T, hk, d, generator=g) * grow).to(dtype).cuda().transpose(1, 2)
             for _ in range(2)]
    if packed:
        kw["cu"] = i32([sum(counts[:i]) for i in range(B + 1)])
    elif lens:
        kw["lens"] = i32(counts)
    ops.kv8_append(pages, scales, *x, table, i32(starts), **kw)
    assert ops.status() == 0
    used = set()
    at = 0
    for b in range(B):
        for kind in range(2):
            if counts[b]:
                rows = x[kind][0][:, at:at + counts[b]] if packed else x[kind][b][:, :counts[b]]
                check_append(before, (pages, scales), rows.double(), table[b], starts[b], counts[b], kind, rope)
        used |= {int(table[b, j]) for j in range(starts[b] // page, per[b])} if counts[b] else set()
        at += counts[b]
    rest = [i for i in range(num) if i not in used]
    assert torch.equal(before[0].view(torch.uint8)[rest], pages.view(torch.uint8)[rest])
    assert torch.equal(before[1][rest].nan_to_num(-1), scales[rest].nan_to_num(-1))
    return pages, scales, table


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("page,d", [(16, 64), (32, 128), (64, 128), (128, 256), (16, 256), (128, 64)])
def test_append_prompts(page, d, dtype):
    for packed in (False, True):
        run_append(page, d, 2, [0, 0, 0], [1, 3 * page + 5, page], dtype, Rope(d), packed, lens=not packed)
        run_append(page, d, 3, [page - 1, 5, 2 * page], [page + 2, 0, 7], dtype, Rope(d // 2, layout="interleaved"), packed,
                   lens=not packed)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_append_one_token(page, dtype):
    """Decode steps: at a page's start, inside it, at its end; small and large enough to raise the scale."""
    for grow in (1.0, 0.01, 50.0):
        run_append(page, 128, 4, [0, 1, page - 1, page, 3 * page + 7], [1] * 5, dtype, Rope(128), grow=grow)
    run_append(page, 256, 1, [page // 2], [1], dtype, Rope(64), grow=20.0)


@pytest.mark.parametrize("R,layout", [(0, "half"), (2, "half"), (10, "half"), (10, "interleaved"), (48, "half"),
                                      (126, "interleaved"), (128, "interleaved")])
def test_append_rotations(R, layout):
    r = Rope(R, layout=layout, scaling={"kind": "yarn", "factor": 4.0, "original": 2048}) if R else None
    run_append(32, 128, 2, [70, 0], [40, 33], BF, r, lens=True)


def test_append_strides():
    """Rows cut out of one projection's output, and offsets that 16-byte accesses do not fit."""
    g = torch.Generator().manual_seed(9)
    for off, dt in ((0, BF), (1, BF), (3, F), (5, HF)):
        rows = torch.randn(2, 21, 2 * 2 * 128 + 9, generator=g).to(dt).cuda()
        k, v = (rows[..., off + i * 256:off + i * 256 + 256].unflatten(-1, (2, 128)).transpose(1, 2) for i in (0, 1))
        run_append(16, 128, 2, [3, 0], [21, 21], dt, Rope(128), x=[k, v])


def test_append_special_values():
    """Zeros give scale 0; infinities saturate, NaN stays, neither sets the scale; tiny and huge values fit."""
    x = torch.randn(2, 1, 20, 64, generator=torch.Generator().manual_seed(3)).cuda()
    for i, edit in enumerate(((0.0, None), (None, float("inf")), (None, float("nan")), (None, -float("inf")), (1e-30, None),
                              (1e30, None), (1e-42, None))):
        k, v = x[:1].clone(), x[1:].clone()
        if edit[0] is not None:
            k *= edit[0]
            v *= edit[0]
        else:
            v[0, 0, 3, 7] = k[0, 0, 18, 63] = edit[1]
        if i == 6:  # below the least scale: all codes are small, none is lost to overflow
            run = run_append(16, 64, 1, [0], [20], F, x=[k, v])
        else:
            run_append(16, 64, 1, [0], [20], F, x=[k, v])
            run_append(16, 64, 1, [21], [20], F, x=[k, v])
    assert run[1].isfinite().any()


def test_append_in_pieces_equals_append_at_once():
    """Where no code gets subnormal the cut into calls leaves the same codes and scales."""
    g = torch.Generator().manual_seed(11)
    k, v = ((torch.rand(1, 2, 75, 128, generator=g) + 0.5) * (1 + torch.arange(75)[:, None] / 20) for _ in range(2))
    k, v, r = k.cuda(), v.cuda(), Rope(32)
    table = i32([[3, 1, 4, 0, 2]])
    got = []
    for cuts in ([75], [1] * 75, [10, 30, 35], [16, 16, 43]):
        pages = torch.zeros(5, 2, 2, 16, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        scales = torch.zeros(5, 2, 2, device="cuda")
        at = 0
        for n in cuts:
            ops.kv8_append(pages, scales, k[:, :, at:at + n], v[:, :, at:at + n], table, i32([at]), turns=r.turns)
            at += n
        got.append((pages.float() * scales[..., None, None], scales))
    for p, s in got[1:]:
        assert torch.equal(s, got[0][1])
        assert torch.equal(p[:, 1], got[0][0][:, 1])  # values
        assert torch.equal(p[:, 0, :, :, 32:], got[0][0][:, 0, :, :, 32:])  # keys past the rotation
    assert ops.status() == 0


def test_append_bad_pages_are_skipped_and_reported():
    pages, scales = pool(4, 1, 16, 64)
    p0 = pages.view(torch.uint8).clone()
    k = torch.randn(2, 1, 40, 64).cuda()
    ops.kv8_append(pages, scales, k, k, i32([[1, 4, 2], [-1, 0, 1 << 30]]), i32([0, 0]), lens=i32([40, 20]))
    assert ops.status() != 0 and ops.status() == 0
    assert torch.equal(pages.view(torch.uint8)[3], p0[3])  # page 3 is no one's
    assert scales[1].isfinite().all() and scales[2].isfinite().all() and scales[0].isfinite().all()
    ops.kv8_append(pages, scales, k, k, i32([[1], [0]]), i32([0, 0]))  # 40 tokens, a table of one page
    assert ops.status() != 0


# ------------------------------------------------------------------------------------------------ attention


def filled(lens, hk, page, d, seed=0, spread=6):
    """A pool whose visible codes are finite and whose other bytes are anything, scales over a range of powers of two."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lens]
    num = sum(per) + 2
    pages, scales = pool(num, hk, page, d, seed)
    table = tables(per, num, seed)
    for b, n in enumerate(lens):
        for j in range(per[b]):
            m = min(page, n - j * page)
            x = torch.randn(2, hk, m, d, generator=g) * 40
            pages.view(torch.uint8)[int(table[b, j]), :, :, :m] = x.to(torch.float8_e4m3fn).view(torch.uint8).cuda()
            e = torch.randint(-spread - 4, -4, (2, hk), generator=g)
            scales[int(table[b, j])] = (2.0 ** e).cuda()
    return pages, scales, table


def check_attend(o, q, pages, scales, table, lens, scale, causal=True):
    B, Hq, T, D = q.shape
    hk = pages.shape[2]
    G, u = Hq // hk, ref.UNIT[q.dtype]
    for b in range(B):
        seen = [lens[b] - T + 1 + t if causal else lens[b] for t in range(T)]
        for h in range(hk):
            k, v = (ref.held(pages, scales, table[b], lens[b], kind, h) for kind in (0, 1))
            for g in range(G):
                want, mass = ref.attend(q[b, h * G + g], k, v, scale, seen)
                got = o[b, h * G + g].double()
                assert torch.equal(torch.isnan(got), torch.isnan(want)), (b, h, g)
                tol = u * want.abs() + (1e-4 if q.dtype == F else 2.0 ** -9) * mass
                bad = ((got - want).abs() > tol) & ~torch.isnan(want)
                assert not bad.any(), (b, h, g, ((got - want).abs() / tol).nan_to_num(0).max())
    assert ops.status() == 0


def run_attend(lens, Hq, hk, T, page, d, dtype, causal=True, seed=0, spread=6, qs=1.0):
    pages, scales, table = filled(lens, hk, page, d, seed, spread)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(len(lens), T, Hq, d, generator=g) * qs).to(dtype).cuda().transpose(1, 2)
    o = ops.kv8_attend(q, pages, scales, table, i32(lens), d ** -0.5, causal)
    check_attend(o, q, pages, scales, table, lens, d ** -0.5, causal)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("page,d", [(16, 64), (16, 128), (32, 256), (64, 128), (128, 128), (128, 256), (64, 64)])
def test_attend_lengths(page, d, dtype):
    run_attend([1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300], 4, 2, 1, page, d, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("G,T", [(1, 1), (3, 1), (7, 1), (8, 1), (1, 5), (12, 1), (12, 4), (16, 2), (5, 7), (1, 33),
                                 (9, 11), (64, 1)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_rows(G, T, d, dtype):
    """Query rows a KV head from one to more than one pass takes; sequences shorter than the rows leave rows empty."""
    run_attend([200, 3, 0, 70, 1], 2 * G, 2, T, 32, d, dtype)


@pytest.mark.parametrize("page", [16, 128])
def test_attend_uneven_batch(page):
    lens = [(i * 97) % 400 for i in range(40)]
    run_attend(lens, 8, 2, 1, page, 128, BF)
    run_attend(lens, 8, 1, 3, page, 128, BF, causal=False)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_long(d):
    run_attend([5000, 9, 2500], 8, 2, 1, 64, d, BF)
    run_attend([4999], 12, 1, 4, 16, d, HF)


def test_attend_scales_far_apart():
    """Pages whose scales differ by up to 2^30: weights times scales stay in f16's range."""
    run_attend([640], 8, 2, 1, 16, 128, BF, spread=30, qs=0.01)
    run_attend([640], 8, 2, 3, 16, 128, HF, spread=30, qs=0.01)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_attend_zero_scales(dtype):
    """Pages of zeros have scale 0."""
    pages, scales, table = filled([100, 64], 2, 16, 128)
    for b, j in ((0, 0), (0, 6), (1, 0), (1, 1), (1, 2), (1, 3)):
        pages.view(torch.uint8)[int(table[b, j])] = 0
        scales[int(table[b, j])] = 0
    q = torch.randn(2, 4, 2, 128, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    o = ops.kv8_attend(q, pages, scales, table, i32([100, 64]), 0.1)
    check_attend(o, q, pages, scales, table, [100, 64], 0.1)
    assert (o[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("T", [1, 4])
def test_attend_nan_codes(T, dtype):
    """A NaN that is held reaches the rows that see it, in its column (a value) or whole (a key), and no others."""
    for kind in (0, 1):
        for key in (0, 120, 197, 198, 199):
            pages, scales, table = filled([200, 90], 2, 32, 128, seed=key)
            pages.view(torch.uint8)[int(table[0, key // 32]), kind, 1, key % 32, 17] = 0xff
            q = torch.randn(2, 8, T, 128, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
            o = ops.kv8_attend(q, pages, scales, table, i32([200, 90]), 0.1)
            check_attend(o, q, pages, scales, table, [200, 90], 0.1)


def test_attend_query_range():
    """Queries far from 1 in either direction (the scale makes up for it), in bf16's range and not f16's."""
    for s in (2.0 ** -60, 2.0 ** 40):
        pages, scales, table = filled([150], 1, 16, 128)
        q = (torch.randn(1, 4, 1, 128, generator=torch.Generator().manual_seed(8)) * s).to(BF).cuda()
        o = ops.kv8_attend(q, pages, scales, table, i32([150]), 0.1 / s)
        check_attend(o, q, pages, scales, table, [150], 0.1 / s)


def test_attend_strides_and_out():
    pages, scales, table = filled([77, 130], 2, 16, 64)
    g = torch.Generator().manual_seed(4)
    for off in (0, 3):
        q = torch.randn(2, 3, 4 * 64 + 11, generator=g).to(BF).cuda()[..., off:off + 256].unflatten(-1, (4, 64)).transpose(1, 2)
        wide = torch.full((2, 3, 4, 64 + 5), 3.0, dtype=BF, device="cuda")
        out = wide[..., off:off + 64].transpose(1, 2)
        assert ops.kv8_attend(q, pages, scales, table, i32([77, 130]), 0.1, out=out) is out
        check_attend(out, q, pages, scales, table, [77, 130], 0.1)
        assert (wide[..., :off] == 3).all() and (wide[..., off + 64:] == 3).all()


def test_attend_bad_page_is_reported():
    pages, scales, table = filled([50], 1, 16, 64)
    q = torch.randn(1, 2, 1, 64, device="cuda").to(BF)
    table[0, 1] = pages.shape[0]
    ops.kv8_attend(q, pages, scales, table, i32([50]), 0.1)
    assert ops.status() != 0 and ops.status() == 0


def test_attend_lengths_out_of_range_are_reported():
    pages, scales, table = filled([50, 30], 1, 16, 64)
    for dt in (BF, F):
        q = torch.randn(2, 2, 1, 64, generator=torch.Generator().manual_seed(1)).to(dt).cuda()
        o = ops.kv8_attend(q, pages, scales, table, i32([50, -3]), 0.1)
        assert ops.status() != 0 and ops.status() == 0
        assert (o[1] == 0).all()
        ops.kv8_attend(q, pages, scales, table[:1].repeat(2, 1), i32([50, 65]), 0.1)
        assert ops.status() != 0
        check_attend(ops.kv8_attend(q, pages, scales, table, i32([50, 30]), 0.1), q, pages, scales, table, [50, 30], 0.1)


@pytest.mark.parametrize("scale", [0.0, -0.07])
def test_attend_any_scale(scale):
    pages, scales, table = filled([90], 1, 16, 128)
    q = torch.randn(1, 4, 2, 128, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    check_attend(ops.kv8_attend(q, pages, scales, table, i32([90]), scale), q, pages, scales, table, [90], scale)


def test_attend_more_sequences_than_a_launch_takes():
    lens = [(i * 7) % 19 for i in range(1500)]
    run_attend(lens, 2, 1, 1, 16, 64, BF)


def test_attend_on_two_streams():
    pages, scales, table = filled([3000, 2000], 2, 16, 128)
    q = torch.randn(2, 8, 1, 128, device="cuda").to(BF)
    n = i32([3000, 2000])
    want = ops.kv8_attend(q, pages, scales, table, n, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([ops.kv8_attend(q, pages, scales, table, n, 0.1) for _ in range(20)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for os in outs for o in os)


def test_attend_in_a_graph():
    """A captured step follows the lengths and the table that it finds at replay."""
    pages, scales, table = filled([500, 400], 2, 16, 128)
    q = torch.randn(2, 8, 1, 128, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    n = i32([500, 400])
    ops.kv8_attend(q, pages, scales, table, n, 0.1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.kv8_attend(q, pages, scales, table, n, 0.1)
    s.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        o = ops.kv8_attend(q, pages, scales, table, n, 0.1)
    n.copy_(i32([33, 399]))
    gr.replay()
    torch.cuda.synchronize()
    check_attend(o, q, pages, scales, table, [33, 399], 0.1)


def test_refused():
    pages, scales, table = filled([20, 20], 2, 16, 64)
    q = torch.zeros(2, 4, 1, 64, dtype=BF, device="cuda")
    k = torch.zeros(2, 2, 1, 64, dtype=BF, device="cuda")
    n = i32([20, 20])
    at, ap = ops.kv8_attend, ops.kv8_append
    for bad in (lambda: at(q[:, :3], pages, scales, table, n, 0.1), lambda: at(q[:1], pages, scales, table, n, 0.1),
                lambda: at(q, pages.view(torch.uint8), scales, table, n, 0.1), lambda: at(q, pages, scales.half(), table, n, 0.1),
                lambda: at(q, pages[:, :, :, :8], scales, table, n, 0.1), lambda: at(q, pages, scales, table.long(), n, 0.1),
                lambda: at(q, pages, scales, table, n[:1], 0.1), lambda: at(q.cpu(), pages, scales, table, n, 0.1),
                lambda: at(q, pages[:, :, :, :8].contiguous(), scales, table, n, 0.1),
                lambda: at(q.double(), pages, scales, table, n, 0.1), lambda: at(q, pages, scales, table, n, float("nan")),
                lambda: ap(pages, scales, k, k[:, :1], table, n), lambda: ap(pages, scales, k, k.half(), table, n),
                lambda: ap(pages, scales, k, k, table[:1], n), lambda: ap(pages, scales, k, k, table, n.long()),
                lambda: ap(pages, scales, k, k, table, n, lens=n, cu=i32([0, 1, 2])),
                lambda: ap(pages, scales, k[:1], k[:1], table, n), lambda: ap(pages, scales, k, k, table, n, cu=i32([0, 1, 2])),
                lambda: ap(pages, scales, k, k, table, n, turns=Rope(128).turns),
                lambda: ap(pages, scales, k.cpu(), k, table, n)):
        with pytest.raises(ValueError):
            bad()


def test_cache_serves_sequences():
    """The whole path through kv8.Cache: prompts packed, decode steps, drafts trimmed, a sequence ended and its pages
    handed out again, against 64-bit attention over what the pages hold, and over the unrounded keys and values within
    e4m3's rounding."""
    g = torch.Generator().manual_seed(21)
    hq, hk, d, page = 8, 2, 128, 16
    c = kv8.Cache(24, page, hk, d)
    r = Rope(d)
    a, b = c.add(), c.add()
    kept = {}

    def go(handles, counts):
        st = c.step(handles, counts)
        rows = sum(counts)
        q, k, v = (torch.randn(1, rows, h, d, generator=g).to(BF).cuda().transpose(1, 2) for h in (hq, hk, hk))
        packed = len(set(counts)) > 1
        if not packed:
            q, k, v = (x[0].unflatten(1, (len(handles), counts[0])).transpose(0, 1) for x in (q, k, v))
        q = r.apply(q, st.positions)
        c.append(st, k, v, rope=r, packed=packed)
        at = 0
        for i, h in enumerate(handles):
            kk, vv = (x[0][:, at:at + counts[i]] if packed else x[i] for x in (k, v))
            pos = torch.arange(c.length(h) - counts[i], c.length(h), device="cuda")
            new = (ref.rotate(kk, pos, r.w), vv.double())
            kept[h] = tuple(torch.cat([o, n], 1) for o, n in zip(kept[h], new)) if h in kept else new
            at += counts[i]
        return st, q

    go([a, b], [37, 20])
    for _ in range(3):
        st, q = go([a, b], [1, 1])
        o = c.attend(st, q, d ** -0.5)
        lens = [c.length(a), c.length(b)]
        check_attend(o, q, c.pages, c.scales, st.table, lens, d ** -0.5)
        for i, h in enumerate((a, b)):
            for x in range(hq):
                k, v = (y[x * hk // hq] for y in kept[h])
                want, mass = ref.attend(q[i, x], k, v, d ** -0.5, [lens[i]])
                # a code is off by 2^-4 of its value at most: keys move scores by up to 2^-4 sum |q k| scale, a few
                # tenths at worst here; values by 2^-4 of themselves
                assert ((o[i, x].double() - want).abs() <= 0.5 * mass + 0.01).all()
    go([a], [4])
    c.trim(a, c.length(a) - 3)
    kept[a] = tuple(x[:, :c.length(a)] for x in kept[a])
    st, q = go([b, a], [4, 4])
    check_attend(c.attend(st, q, d ** -0.5), q, c.pages, c.scales, st.table, [c.length(b), c.length(a)], d ** -0.5)
    free = c.free_pages
    c.drop(b)
    assert c.free_pages == free + -(-27 // page)
    with pytest.raises(ValueError, match="pages needed"):
        c.step([a], [24 * page])
    assert ops.status() == 0
