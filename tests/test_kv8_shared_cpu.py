"""kv8.Cache's shared pages on the host: forks, copies before a write, tokens kept, pools resized. The kernels' calls are stood
in for by forms that move the tokens' names about, so that what each sequence holds can be read back."""
import random

import pytest
import torch

from larder_b200 import kv8

PAGE, HK, D = 16, 2, 64


@pytest.fixture
def names(monkeypatch):
    """Stand-ins of the kernels: a page is a list of token names, kept by the pool's address; `fail` refuses the next call of
    that name; `wrote` lists the pages that appends wrote."""
    mem = {"fail": None, "wrote": [], "pools": {}}

    def pool(pages):
        return mem["pools"].setdefault(pages.data_ptr(), {})

    def may(name):
        if mem["fail"] == name:
            mem["fail"] = None
            raise ValueError(f"{name}: refused")

    def append(pages, scales, k, v, table, start, cu=None, **kw):
        may("append")
        at = pool(pages)
        for b in range(table.shape[0]):
            rows = k[0, 0, int(cu[b]):int(cu[b + 1]), 0] if cu is not None else k[b, 0, :, 0]
            for t, x in enumerate(rows.tolist()):
                p = int(start[b]) + t
                page = int(table[b, p // PAGE])
                at.setdefault(page, [None] * PAGE)[p % PAGE] = x
                mem["wrote"].append(page)

    def copy(pages, scales, src, dst, into=None):
        may("copy")
        at, to = pool(pages), pool(pages if into is None else into[0])
        held = [list(at.get(int(i), [None] * PAGE)) for i in src]
        for i, x in zip(dst.tolist(), held):
            to[i] = x

    def compact(pages, scales, table, keep, cu, to, start, **kw):
        may("compact")
        at = pool(pages)
        read, wrote = set(), set()
        for b in range(table.shape[0]):
            assert int(start[b]) % PAGE == 0
            for i, pos in enumerate(keep[int(cu[b]):int(cu[b + 1])].tolist()):
                new = int(start[b]) + i
                page = int(to[b, new // PAGE])
                if new % PAGE == 0:
                    assert page not in wrote
                read.add(int(table[b, pos // PAGE]))
                wrote.add(page)
                at.setdefault(page, [None] * PAGE)[new % PAGE] = at[int(table[b, pos // PAGE])][pos % PAGE]
        assert not read & wrote

    monkeypatch.setattr(kv8.ops, "kv8_append", append)
    monkeypatch.setattr(kv8.ops, "kv8_copy", copy)
    monkeypatch.setattr(kv8.ops, "kv8_compact", compact)
    monkeypatch.setattr(kv8.ops, "kv8_attend", lambda *a: "o")
    monkeypatch.setattr(kv8.ops, "kv8_attend_packed", lambda *a: "packed")
    return mem


def make(num=12):
    return kv8.Cache(num, PAGE, HK, D, device="cpu")


def put(cache, handles, tokens):
    """Appends named tokens, packed; returns the step."""
    step = cache.step(handles, [len(t) for t in tokens])
    flat = [x for t in tokens for x in t]
    k = torch.tensor(flat, dtype=torch.float64).view(1, 1, -1, 1).expand(1, HK, len(flat), D)
    cache.append(step, k, k, packed=True)
    return step


def held(mem, cache, handle):
    ids, n = cache._seqs[handle]
    at = mem["pools"].get(cache.pages.data_ptr(), {})
    return [at[ids[p // PAGE]][p % PAGE] for p in range(n)]


def whole(cache):
    """The page counts are what the sequences say, and every page is free or held."""
    refs = [0] * len(cache._refs)
    for ids, n in cache._seqs.values():
        assert len(ids) == -(-n // PAGE)
        for i in ids:
            refs[i] += 1
    assert refs == cache._refs
    assert sorted(cache._free) == [i for i, r in enumerate(refs) if r == 0]


def test_fork_shares_until_a_write(names):
    c = make()
    a = c.add()
    put(c, [a], [range(40)])
    b = c.fork(a)
    assert c.free_pages == 9 and c.length(b) == 40 and held(names, c, b) == list(range(40))
    put(c, [b], [[100]])  # the third page, half filled, is copied for b
    assert c.free_pages == 8
    assert held(names, c, b) == list(range(40)) + [100] and held(names, c, a) == list(range(40))
    put(c, [a], [[200, 201]])  # a holds its page alone again: no copy
    assert c.free_pages == 8
    assert held(names, c, a) == list(range(40)) + [200, 201] and held(names, c, b) == list(range(40)) + [100]
    d = c.fork(a, 32)  # at a page's end: nothing to copy
    put(c, [d], [[300]])
    assert c.free_pages == 7 and held(names, c, d) == list(range(32)) + [300]
    e = c.fork(a, 35)
    put(c, [a, e], [[202], [400]])  # both in one step, one of them keeps the page
    assert held(names, c, a) == list(range(40)) + [200, 201, 202] and held(names, c, e) == list(range(35)) + [400]
    assert c.length(c.fork(a, 0)) == 0
    for h in (a, b, d):
        c.drop(h)
    whole(c)
    assert held(names, c, e) == list(range(35)) + [400]


def test_three_that_share_in_one_step(names):
    c = make()
    a = c.add()
    put(c, [a], [range(5)])
    b, d = c.fork(a), c.fork(a)
    put(c, [b, d, a], [[10], [20], [30]])
    assert [held(names, c, h)[5:] for h in (a, b, d)] == [[30], [10], [20]] and c.free_pages == 9
    whole(c)


def test_step_counts_the_copies_it_needs(names):
    c = make(2)
    a = c.add()
    put(c, [a], [range(20)])
    b = c.fork(a)
    with pytest.raises(ValueError, match="1 pages needed, 0 free"):
        c.step([b], [1])
    whole(c)
    assert c.length(b) == 20
    c.drop(a)
    put(c, [b], [[7]])
    assert held(names, c, b) == list(range(20)) + [7]


def test_a_refused_copy_leaves_the_pool_as_it_was(names):
    c = make()
    a = c.add()
    put(c, [a], [range(20)])
    b, d = c.fork(a), c.fork(a)
    names["fail"] = "copy"
    before = [list(c._seqs[h][0]) for h in (a, b, d)]
    with pytest.raises(ValueError, match="refused"):
        c.step([b, d, a], [1, 30, 2])
    assert [c._seqs[h][0] for h in (a, b, d)] == before and c.free_pages == 10
    whole(c)
    put(c, [b, d, a], [[1], range(30), [3, 4]])  # nothing was reserved
    assert held(names, c, b) == list(range(20)) + [1]


def test_no_fork_of_tokens_not_appended(names):
    c = make()
    a = c.add()
    put(c, [a], [range(10)])
    step = c.step([a], [3])
    with pytest.raises(ValueError, match="not appended"):
        c.fork(a)
    with pytest.raises(ValueError, match="not appended"):
        c.keep([a], [[1]])
    with pytest.raises(ValueError, match="not appended"):
        c.resize(20)
    b = c.fork(a, 10)  # those before are
    assert held(names, c, b) == list(range(10))
    # the page of the reserved tokens is shared now: an append into it would change b
    k = torch.zeros(1, HK, 3, D)
    with pytest.raises(ValueError, match="shares the pages"):
        c.append(step, k, k)
    c.trim(a, 10)
    put(c, [a], [[5]])
    assert held(names, c, b) == list(range(10)) and held(names, c, a) == list(range(10)) + [5]


def test_keep(names):
    c = make()
    a, b = c.add(), c.add()
    put(c, [a, b], [range(50), range(100, 130)])
    f = c.fork(a)
    c.keep([a, b], [list(range(20)) + [30, 40, 49], [5, 6]])
    assert held(names, c, a) == list(range(20)) + [30, 40, 49] and held(names, c, b) == [105, 106]
    assert held(names, c, f) == list(range(50))
    assert c._seqs[a][0][0] == c._seqs[f][0][0] and c._refs[c._seqs[a][0][0]] == 2  # the first page stays where it is
    whole(c)
    c.keep([a, b], [range(7), []])  # nothing moves
    assert held(names, c, a) == list(range(7)) and c.length(b) == 0
    whole(c)
    put(c, [a], [[9]])
    assert held(names, c, a) == list(range(7)) + [9] and held(names, c, f) == list(range(50))


@pytest.mark.parametrize("at", [[3, 3], [4, 2], [-1, 2], [0, 50]])
def test_keep_refuses_bad_positions(names, at):
    c = make()
    a, b = c.add(), c.add()
    put(c, [a, b], [range(50), range(30)])
    with pytest.raises(ValueError, match="positions"):
        c.keep([b, a], [[1], at])
    assert c.length(a) == 50 and c.length(b) == 30
    for bad in (([a, a], [[1], [2]]), ([a], [[1], [2]])):
        with pytest.raises(ValueError, match="distinct"):
            c.keep(*bad)


def test_keep_refused_for_want_of_pages_or_by_the_kernel(names):
    c = make(4)
    a = c.add()
    put(c, [a], [range(60)])
    with pytest.raises(ValueError, match="1 pages needed, 0 free"):
        c.keep([a], [[3, 5]])
    assert held(names, c, a) == list(range(60))
    c.trim(a, 40)
    names["fail"] = "compact"
    with pytest.raises(ValueError, match="refused"):
        c.keep([a], [[3, 5]])
    whole(c)
    c.keep([a], [[3, 5]])
    assert held(names, c, a) == [3, 5] and c.free_pages == 3


def test_resize(names):
    c = make()
    a, b = c.add(), c.add()
    put(c, [a, b], [range(40), range(100, 120)])
    f = c.fork(b)
    c.drop(a)
    with pytest.raises(ValueError, match="do not fit"):
        c.resize(1)
    c.resize(2)
    assert c.free_pages == 0 and c.pages.shape[0] == 2 and held(names, c, b) == held(names, c, f) == list(range(100, 120))
    whole(c)
    c.resize(7)
    put(c, [b], [[1]])
    assert held(names, c, b) == list(range(100, 120)) + [1] and held(names, c, f) == list(range(100, 120))
    whole(c)


def test_steps_made_before_a_move_are_refused(names):
    c = make()
    a, b = c.add(), c.add()
    s = put(c, [a, b], [range(20), range(20)])
    alone = c.step([b], [0])
    q, k = torch.zeros(2, HK, 1, D), torch.zeros(1, HK, 40, D)
    assert c.attend(s, q, 1.0) == "o"
    c.keep([a], [[1, 3]])
    for call in (lambda: c.attend(s, q, 1.0), lambda: c.append(s, k, k, packed=True)):
        with pytest.raises(ValueError, match="moved"):
            call()
    assert c.attend(alone, q[:1], 1.0) == "o"  # the other sequence's
    f = c.fork(b)
    assert c.attend(alone, q[:1], 1.0) == "o"
    put(c, [b], [[5]])  # b's page is copied for it
    with pytest.raises(ValueError, match="moved"):
        c.attend(alone, q[:1], 1.0)
    late = c.step([a, b, f], [0, 0, 0])
    c.resize(12)
    with pytest.raises(ValueError, match="moved"):
        c.attend(late, q, 1.0)
    assert c.attend(c.step([a, b], [0, 0]), q, 1.0) == "o"


def test_packed_attend(names):
    c = make()
    a, b = c.add(), c.add()
    s = put(c, [a, b], [range(5), range(3)])
    assert c.attend(s, torch.zeros(1, 4, 8, D), 1.0, packed=True) == "packed"
    with pytest.raises(ValueError, match="8 packed rows"):
        c.attend(s, torch.zeros(1, 4, 7, D), 1.0, packed=True)


@pytest.mark.parametrize("seed", range(8))
def test_any_order_of_calls(names, seed):
    """Random forks, appends, trims, cuts, drops and resizes: every sequence holds what a list of its tokens says, and no
    append writes a page that two sequences hold."""
    rng = random.Random(seed)
    c = make(24)
    want, fresh = {c.add(): []}, iter(range(10 ** 6))
    for _ in range(300):
        what = rng.choice(["fork", "put", "put", "put", "trim", "keep", "drop", "resize", "add"])
        h = rng.choice(list(want)) if want else None
        try:
            if what == "add" or h is None:
                want[c.add()] = []
            elif what == "fork":
                n = rng.choice([None, rng.randint(0, len(want[h]))])
                want[c.fork(h, n)] = list(want[h][:n])
            elif what == "put":
                hs = rng.sample(list(want), rng.randint(1, min(4, len(want))))
                new = [[next(fresh) for _ in range(rng.choice([0, 1, 1, 5, 20]))] for _ in hs]
                names["wrote"].clear()
                put(c, hs, new)
                for x, t in zip(hs, new):
                    want[x] += t
                assert all(c._refs[i] == 1 for i in names["wrote"])
            elif what == "trim":
                n = rng.randint(0, len(want[h]))
                c.trim(h, n)
                del want[h][n:]
            elif what == "keep":
                at = sorted(rng.sample(range(len(want[h])), rng.randint(0, len(want[h]))))
                c.keep([h], [at])
                want[h] = [want[h][i] for i in at]
            elif what == "drop":
                c.drop(h)
                del want[h]
            else:
                c.resize(rng.randint(18, 30))
        except ValueError as e:
            assert "free" in str(e) or "fit" in str(e), e
        whole(c)
        for x, t in want.items():
            assert held(names, c, x) == t


def test_cpu_tensors_are_refused():
    pages = torch.zeros(4, 2, HK, PAGE, D, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales, table = torch.zeros(4, 2, HK), torch.zeros(1, 2, dtype=torch.int32)
    n, cu = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(1, 4, 3, D, dtype=torch.bfloat16)
    for call in (lambda: kv8.ops.kv8_attend_packed(q, pages, scales, table, n, cu, 0.1),
                 lambda: kv8.ops.kv8_copy(pages, scales, n, n),
                 lambda: kv8.ops.kv8_copy(pages, scales, n, n, into=(pages.clone(), scales.clone())),
                 lambda: kv8.ops.kv8_compact(pages, scales, table, n, cu, table, n)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_keep_takes_any_iterable_of_positions(names):
    c = make()
    a, b = c.add(), c.add()
    put(c, [a, b], [range(40), range(100, 140)])
    c.keep([a, b], [iter([3, 4]), (i for i in range(2))])
    assert held(names, c, a) == [3, 4] and held(names, c, b) == [100, 101]
    with pytest.raises(TypeError):
        c.keep([a, b], [[1], 5])
    assert c.length(a) == c.length(b) == 2
