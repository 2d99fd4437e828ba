"""Copying pages of the paged 8-bit cache and compacting its sequences, against 64 bits.

A copy is exact. A compacted page's scale is the least power of two s with max |x| <= 448 s over its held values, and its codes
the nearest to x / s: exactly for values and for keys that are not turned (code * s is exact in fp32, and so is a division by a
power of two), within half a code step plus the turned value's own error otherwise: fp32 rotation by an angle exact to 2^-24
turns, under 2^-18 (|x0| + |x1|), which may also lift a maximum over 448 s."""
import pytest
import torch

from larder_b200 import kv8, ops
from larder_b200.rope import Rope

import serve_ref as ref
from test_gpu_kv8_chunk import cache, close, expect, i32, queries, starts

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def pool(num, hk, page, d, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(0, 256, (num, 2, hk, page, d), generator=g, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            torch.rand(num, 2, hk, generator=g, device="cuda"))


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("n", [0, 1, 2, 5, 333])
@pytest.mark.parametrize("hk,page,d", [(1, 16, 64), (2, 64, 128), (8, 32, 128), (3, 128, 256), (5, 16, 64)])
def test_copy(hk, page, d, n):
    """Within a pool and into another one; every other page stays as it is."""
    pages, scales = pool(2 * n + 3, hk, page, d)
    ids = torch.randperm(2 * n + 3, generator=torch.Generator().manual_seed(n)).int().cuda()
    src, dst = ids[:n].contiguous(), ids[n:2 * n].contiguous()
    p, s = pages.clone(), scales.clone()
    ops.kv8_copy(p, s, src, dst)
    want_p, want_s = pages.view(torch.uint8).clone(), scales.clone()
    want_p[dst.long()], want_s[dst.long()] = want_p[src.long()], want_s[src.long()]
    assert same(p, want_p) and torch.equal(s, want_s) and ops.status() == 0
    other, more = pool(n + 2, hk, page, d, seed=1)
    want_p, want_s = other.view(torch.uint8).clone(), more.clone()
    into = torch.randperm(n + 2, generator=torch.Generator().manual_seed(n)).int().cuda()[:n].contiguous()
    want_p[into.long()], want_s[into.long()] = pages.view(torch.uint8)[src.long()], scales[src.long()]
    ops.kv8_copy(pages, scales, src, into, into=(other, more))
    assert same(other, want_p) and torch.equal(more, want_s) and ops.status() == 0


def test_copy_one_page_to_many_and_to_itself():
    pages, scales = pool(9, 2, 16, 128)
    p, s = pages.clone(), scales.clone()
    ops.kv8_copy(p, s, i32([4, 4, 4, 7]), i32([0, 8, 2, 7]))
    want = torch.arange(9)
    want[[0, 8, 2]] = 4
    assert same(p, pages.view(torch.uint8)[want.cuda()]) and torch.equal(s, scales[want.cuda()]) and ops.status() == 0


def test_copy_skips_and_reports_bad_ids():
    pages, scales = pool(9, 2, 16, 64)
    for src, dst in (([1, 9], [2, 3]), ([1, -1], [2, 3]), ([1, 3], [2, 9]), ([1, 3], [2, -5]), ([1, 1 << 30], [2, 1 << 30])):
        p, s = pages.clone(), scales.clone()
        ops.kv8_copy(p, s, i32(src), i32(dst))
        want = torch.arange(9)
        want[2] = 1
        assert same(p, pages.view(torch.uint8)[want.cuda()]) and torch.equal(s, scales[want.cuda()])
        assert ops.status() != 0 and ops.status() == 0
    small = pool(2, 2, 16, 64, seed=1)
    ops.kv8_copy(pages, scales, i32([0, 8]), i32([1, 2]), into=small)  # the other pool's bounds
    assert ops.status() != 0 and same(small[0][1], pages[0])


def test_copy_past_32_bits():
    num = (1 << 32) // (2 * 8 * 128 * 256) + 3
    pages, scales = pool(4, 8, 128, 256)
    big = torch.zeros(num, 2, 8, 128, 256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    more = torch.zeros(num, 2, 8, device="cuda")
    ops.kv8_copy(pages, scales, i32([1, 2]), i32([num - 1, 0]), into=(big, more))
    ops.kv8_copy(big, more, i32([num - 1]), i32([num - 2]))
    for i in (num - 1, num - 2):
        assert same(big[i], pages[1]) and torch.equal(more[i], scales[1])
    assert same(big[0], pages[2]) and ops.status() == 0


def test_copy_refusals():
    pages, scales = pool(6, 2, 16, 64)
    a, b = i32([1]), i32([2])
    wide, less = pool(6, 2, 16, 128), pool(6, 1, 16, 64)
    for bad in ((pages[:, :, :, ::2], scales, a, b), (pages, scales[1:], a, b), (pages, scales.double(), a, b),
                (pages, scales, a.long(), b), (pages, scales, a, i32([1, 2])), (pages, scales, a.cpu(), b),
                (pages.cpu(), scales.cpu(), a, b), (pages.view(torch.uint8), scales, a, b), (pages, scales, a, b, wide),
                (pages, scales, a, b, less), (pages, scales, a, b, (pages, scales.cpu())), (pages[0], scales, a, b)):
        with pytest.raises(ValueError):
            ops.kv8_copy(*bad)
    with pytest.raises(ValueError):
        ops.kv8_copy(pages[..., :16, :48].contiguous(), scales, a, b)
    assert ops.status() == 0


def check_compact(before, after, table, keeps, to, start, rope):
    (p0, s0), (p1, s1) = before, after
    page, D = p0.shape[3:]
    u0, u1 = p0.view(torch.uint8), p1.view(torch.uint8)
    used = set()
    for b, at in enumerate(keeps):
        at = torch.tensor(at, dtype=torch.long, device="cuda")
        for j in range(-(-len(at) // page)):
            rows = at[j * page:(j + 1) * page]
            n, pg = len(rows), int(to[b, start[b] // page + j])
            used.add(pg)
            ids = table[b].long()[rows // page]
            for kind in (0, 1):
                for h in range(p0.shape[2]):
                    c = u0[ids, kind, h, rows % page].view(torch.float8_e4m3fn).double()
                    x = c * s0[ids, kind, h].double()[:, None]
                    slack = torch.zeros_like(x)
                    if kind == 0 and rope is not None:
                        turn = torch.arange(n, device="cuda") + start[b] + j * page - rows
                        slack = 2.0 ** -18 * ref.pair_sum(x, rope.dims, rope.layout)
                        slack[:, rope.dims:] = 0
                        x = ref.rotate(x, turn, rope.w, rope.layout)
                    fin = torch.isfinite(x)
                    top = x[fin].abs().max() if fin.any() else torch.zeros((), dtype=torch.float64)
                    up = float(slack[fin].max()) if fin.any() else 0.0
                    now = float(s1[pg, kind, h])
                    assert now in {ref.scale_of(float(top)), ref.scale_of(float(top) + up), ref.scale_of(max(float(top) - up, 0.0))}
                    got = p1[pg, kind, h, :n].double()
                    assert torch.equal(torch.isnan(got), torch.isnan(x))
                    z = x / now if now else torch.zeros_like(x)
                    err = (got - z.clamp(-448, 448)).abs()
                    assert (err <= ref.half_step(z.clamp(-448, 448)) + (slack / now if now else 0))[fin].all()
                    assert torch.equal(u0[pg, kind, h, n:], u1[pg, kind, h, n:])  # past the last token
    rest = [i for i in range(p0.shape[0]) if i not in used]
    assert torch.equal(u0[rest], u1[rest]) and torch.equal(s0[rest].nan_to_num(-1), s1[rest].nan_to_num(-1))


def run_compact(lens, keeps, start, hk, page, d, rope=None, seed=0, spread=1.5, edit=None):
    """keeps[b]: old positions of the tokens that become positions start[b] on of sequence b."""
    need = [-(-len(k) // page) for k in keeps]
    per = [-(-n // page) for n in lens]
    num = sum(per) + sum(need) + 2
    pages, scales, table = cache(lens, hk, page, d, seed, spread, num)
    if edit:
        edit(pages, scales, table)
    free = [i for i in range(num) if i not in set(table.flatten().tolist())]
    to = torch.full((len(lens), max(s // page + n for s, n in zip(start, need)) or 1), 1 << 30, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            to[b, start[b] // page + j] = free.pop()
    to = to.cuda()
    before = pages.clone(), scales.clone()
    kw = {} if rope is None else {"turns": rope.turns, "layout": rope.layout}
    ops.kv8_compact(pages, scales, table, i32([x for k in keeps for x in k]), i32(starts([len(k) for k in keeps])), to,
                    i32(start), **kw)
    assert ops.status() == 0
    check_compact(before, (pages, scales), table, keeps, to, start, rope)
    return pages, scales, table, to


@pytest.mark.parametrize("layout", [None, "half", "interleaved"])
@pytest.mark.parametrize("hk,page,d", [(2, 16, 64), (1, 16, 128), (2, 32, 128), (3, 64, 128), (1, 128, 128), (2, 128, 256),
                                       (1, 16, 256), (1, 128, 64), (8, 16, 64)])
def test_compact(hk, page, d, layout):
    """Windows, scattered tokens, one token, none, behind pages that stay."""
    g = torch.Generator().manual_seed(d + page)
    lens = [5 * page + 3, 2 * page, page + 1, 3 * page, 4]
    some = sorted(torch.randperm(lens[0], generator=g)[:2 * page + 5].tolist())
    keeps = [some, list(range(page + 7, 2 * page)), [], list(range(page + 3, 3 * page)), [2]]
    start = [0, 0, page, page, 0]
    for R in (d, d // 2):
        run_compact(lens, keeps, start, hk, page, d, None if layout is None else Rope(R, layout=layout))


@pytest.mark.parametrize("R,layout", [(2, "half"), (10, "half"), (10, "interleaved"), (48, "half"), (62, "interleaved"),
                                      (16, "half"), (120, "half")])
def test_compact_odd_rotations(R, layout):
    run_compact([100, 40], [list(range(3, 90, 2)), [39, 1, 1, 0]], [0, 16], 2, 16, 128, Rope(R, layout=layout))


def test_compact_any_order_and_twice():
    """Positions in any order, the same one twice, and a scaled rotation's angles at far positions."""
    rope = Rope(128, base=1e6, scaling={"kind": "yarn", "factor": 4.0, "original": 32768})
    keep = [60000, 3, 3, 59999, 0, 41234] + list(range(50000, 50100))
    pages, scales, table = cache([60001], 1, 128, 128, num=480)
    free = sorted(set(range(480)) - set(table.flatten().tolist()))
    to = i32([free[:1]])
    before = pages.clone(), scales.clone()
    ops.kv8_compact(pages, scales, table, i32(keep), i32([0, len(keep)]), to, i32([0]), turns=rope.turns)
    check_compact(before, (pages, scales), table, [keep], to, [0], rope)


def test_compact_nan_zero_and_loud_codes():
    """NaN codes stay NaN and do not set the scale; pages of zeros; scales far apart; codes at the end of the range."""
    def edit(pages, scales, table):
        raw = pages.view(torch.uint8)
        ids = table[0].long()
        raw[ids[0], :, :, 3, 5] = 0x7F
        raw[ids[1], :, :, 2] = 0xFF
        raw[ids[2]], scales[ids[2]] = 0, 0.0
        raw[ids[3]], scales[ids[3]] = 0, 0.0
        raw[ids[4], 0, :, 1, 9] = 0x7E  # 448
        scales[ids[5]] = 2.0 ** -126
        scales[ids[6]] = 2.0 ** 100
        raw[ids[7]] = 0x01  # the least subnormal
    for rope in (None, Rope(64), Rope(32, layout="interleaved")):
        run_compact([9 * 16], [list(range(2, 40)) + list(range(50, 96)) + [100, 101] + list(range(112, 144))], [0], 2, 16, 64,
                    rope, edit=edit)
        run_compact([9 * 16], [list(range(33, 63))], [0], 2, 16, 64, rope, edit=edit)  # zeros only
        run_compact([9 * 16], [list(range(18, 19))], [0], 2, 16, 64, rope, edit=edit)  # NaN only


def test_compact_is_the_append_of_the_held_values():
    """The codes that append leaves in fresh pages for the held values."""
    lens, keep = [700], sorted(torch.randperm(700, generator=torch.Generator().manual_seed(1))[:301].tolist())
    pages, scales, table, to = run_compact(lens, [keep], [0], 2, 32, 128)
    at = torch.tensor(keep).cuda()
    k, v = (torch.stack([ref.held(pages, scales, table[0], 700, i, h)[at] for h in range(2)])[None].float() for i in (0, 1))
    p, s = pages.clone(), torch.zeros_like(scales)
    ops.kv8_append(p, s, k, v, to, i32([0]))
    ids = to[0].long()
    assert torch.equal(s[ids], scales[ids]) and same(p, pages)


def test_compact_reports_what_it_skips():
    for rope in (None, Rope(64), Rope(10)):
        kw = {} if rope is None else {"turns": rope.turns}
        pages, scales, table = cache([100, 50], 2, 16, 64, num=20)
        free = sorted(set(range(20)) - set(table.flatten().tolist()))
        to, keep, cu = i32([free[:2], free[2:4]]), i32(list(range(40, 60)) + list(range(20))), i32([0, 20, 40])
        p, s = pages.clone(), scales.clone()
        ops.kv8_compact(p, s, table, keep, cu, to, i32([0, 0]), **kw)
        assert ops.status() == 0
        second = to[1].long()

        def run(**bad):
            a = {"table": table, "keep": keep, "cu": cu, "to": to, "start": i32([0, 0]), **bad}
            x, y = pages.clone(), scales.clone()
            ops.kv8_compact(x, y, a["table"], a["keep"], a["cu"], a["to"], a["start"], **kw)
            assert ops.status() != 0 and ops.status() == 0
            return x, y

        for bad in (-1, 1 << 30, 20):
            t, u = table.clone(), to.clone()
            t[0, 2], u[0, 1] = bad, bad
            for x, y in (run(table=t), run(to=u)):
                assert same(x[second], p[second]) and torch.equal(y[second], s[second])
            k = keep.clone()
            k[3] = bad if bad != 20 else 16 * table.shape[1]
            x, y = run(keep=k)
            assert same(x[second], p[second]) and (x.view(torch.uint8)[to[0, 0].long(), 1, :, 3] == 0).all()
        run(start=i32([8, 0])), run(start=i32([-16, 0])), run(start=i32([32, 0]))
        for c in ([-1, 20, 40], [0, 20, 41], [0, 30, 20], [1 << 30, 20, -(1 << 30)]):
            run(cu=i32(c))


def test_compact_in_a_graph_and_on_another_stream():
    lens, keeps = [300, 90], [list(range(7, 250, 2)), list(range(30, 90))]
    pages, scales, table = cache(lens, 2, 32, 128, num=40)
    free = sorted(set(range(40)) - set(table.flatten().tolist()))
    to = i32([free[:4], free[4:8]])
    rope = Rope(128)
    args = (table, i32(sum(keeps, [])), i32([0, len(keeps[0]), len(keeps[0]) + 60]), to, i32([0, 0]), rope.turns)
    p, s = pages.clone(), scales.clone()
    ops.kv8_compact(p, s, *args)
    x, y = pages.clone(), scales.clone()
    x2, y2 = pages.clone(), scales.clone()
    src, dst = to[0].contiguous(), i32(free[8:12])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv8_compact(x, y, *args)
        ops.kv8_copy(x, y, src, dst)
    x.view(torch.uint8).copy_(pages.view(torch.uint8)), y.copy_(scales)
    g.replay()
    assert same(x[to.flatten().long()], p[to.flatten().long()]) and same(x[dst.long()], p[src.long()])
    assert torch.equal(y[dst.long()], s[src.long()])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        ops.kv8_compact(x2, y2, *args)
    torch.cuda.synchronize()
    assert same(x2, p) and torch.equal(y2.nan_to_num(-1), s.nan_to_num(-1)) and ops.status() == 0


def test_compact_refusals():
    pages, scales, table = cache([100], 2, 16, 64)
    keep, cu, to, start = i32([1, 2]), i32([0, 2]), i32([[8]]), i32([0])
    turns = Rope(64).turns

    def call(**kw):
        a = {"pages": pages, "scales": scales, "table": table, "keep": keep, "cu": cu, "to": to, "start": start, **kw}
        ops.kv8_compact(**a)

    call()
    for bad in ({"keep": keep.long()}, {"keep": keep.cpu()}, {"cu": i32([0])}, {"cu": cu.float()}, {"to": to[0]},
                {"to": i32([[1], [2]])}, {"to": to.long()}, {"start": i32([0, 0])}, {"turns": turns.int()},
                {"turns": Rope(128).turns}, {"turns": turns, "layout": "other"}, {"pages": pages[:, :1]},
                {"scales": scales.half()}, {"table": table.t()[:1]}, {"pages": pages.cpu(), "scales": scales.cpu()}):
        with pytest.raises(ValueError):
            call(**bad)
    assert ops.status() == 0


def test_shared_cache_end_to_end():
    """Two sequences forked from one prompt, continued in uneven chunks, one of them cut to a window, the pool made smaller:
    attention over each is that over the tokens it should hold."""
    hk, d, page = 2, 128, 32
    rope = Rope(d)
    c = kv8.Cache(64, page, hk, d)
    kv = {s: [queries(hk, 300, d, BF, seed=10 + s + i)[0] for i in (0, 4)] for s in range(3)}

    def put(handles, tokens):
        """tokens[i]: (source, first, last) of the new tokens of handles[i]."""
        k, v = (torch.cat([kv[s][i][:, a:b] for s, a, b in tokens], 1)[None] for i in (0, 1))
        step = c.step(handles, [b - a for _, a, b in tokens])
        c.append(step, k, v, rope=rope, packed=True)
        return step

    a = c.add()
    put([a], [(0, 0, 170)])
    b = c.fork(a)
    step = put([a, b], [(1, 0, 3), (2, 0, 90)])
    held = {a: [(0, i) for i in range(170)] + [(1, i) for i in range(3)],
            b: [(0, i) for i in range(170)] + [(2, i) for i in range(90)]}

    def check(handles, counts, step, window=None):
        T = sum(counts)
        q = queries(4, T, d, BF, seed=50)
        o = c.attend(step, q, 0.1, packed=True)
        at = 0
        for h, n in zip(handles, counts):
            L = c.length(h)
            for hh in range(4):
                k = torch.stack([kv[s][0][hh // 2, i] for s, i in held[h]])
                v = torch.stack([kv[s][1][hh // 2, i] for s, i in held[h]]).double()
                k = ref.rotate(k, torch.arange(L, device="cuda"), rope.w)
                s = q[0, hh, at:at + n].double() @ k.T * 0.1
                s = s.masked_fill(torch.arange(L, device="cuda") >= (L - n + 1 + torch.arange(n, device="cuda"))[:, None], -1e30)
                want = torch.softmax(s, -1) @ v
                # each code is off by 2^-4 of its value at most (twice after a cut), at random: 10 % of the norm is ample
                assert (o[0, hh, at:at + n].double() - want).norm() <= 0.1 * want.norm()
            at += n
        close(o, *expect(q, c.pages, c.scales, step.table, [c.length(h) for h in handles], counts, 0.1), BF)

    check([a, b], [3, 90], step)
    window = list(range(4)) + list(range(150, 260))
    c.keep([b], [window], rope)
    held[b] = [held[b][i] for i in window]
    step = put([b, a], [(2, 90, 120), (1, 3, 4)])
    held[b] += [(2, i) for i in range(90, 120)]
    held[a] += [(1, 3)]
    check([b, a], [30, 1], step)
    c.resize(16)
    step = put([a, b], [(1, 4, 6), (2, 120, 121)])
    held[a] += [(1, 4), (1, 5)]
    held[b] += [(2, 120)]
    check([a, b], [2, 1], step)
    assert ops.status() == 0
