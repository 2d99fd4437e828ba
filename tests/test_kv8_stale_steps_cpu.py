"""kv8.Cache on the host, steps that what happened since has overtaken: which appends and attends are refused, and that none of
them reaches pages or tokens that are not the step's."""
import random

import pytest
import torch

from larder_b200 import kv8

from test_kv8_shared_cpu import D, HK, PAGE, held, make, names, put, whole  # noqa: F401 (names: the kernels' stand-ins)


def rows(n):
    return torch.full((1, HK, n, D), -1.0)


def q(B=1):
    return torch.zeros(B, 4, 1, D)


def test_no_attention_over_tokens_whose_append_was_refused_for_a_shared_page(names):
    c = make()
    a = c.add()
    put(c, [a], [range(10)])
    s = c.step([a], [3])
    b = c.fork(a, 10)
    with pytest.raises(ValueError, match="shares the pages"):
        c.append(s, rows(3), rows(3))
    with pytest.raises(ValueError, match="not appended"):
        c.attend(s, q(), 1.0)
    later = put(c, [a], [[7]])  # in a page of a's own, behind the three that are not there
    with pytest.raises(ValueError, match="not appended"):
        c.attend(later, q(), 1.0)
    assert held(names, c, b) == list(range(10)) and c.attend(c.step([b], [0]), q(), 1.0) == "o"
    c.trim(a, 10)
    assert c.attend(put(c, [a], [[5]]), q(), 1.0) == "o" and held(names, c, a) == list(range(10)) + [5]


def test_no_attention_over_tokens_whose_append_was_refused_for_a_moved_page(names):
    c = make()
    a = c.add()
    put(c, [a], [range(10)])
    s = c.step([a], [3])
    b = c.fork(a, 10)
    later = put(c, [a], [[7]])  # the page is copied for a
    with pytest.raises(ValueError, match="moved"):
        c.append(s, rows(3), rows(3))
    for step in (later, c.step([a], [0])):
        with pytest.raises(ValueError, match="not appended"):
            c.attend(step, q(), 1.0)
    c.drop(b)
    c.trim(a, 10)
    assert c.attend(put(c, [a], [[5]]), q(), 1.0) == "o"


def test_a_refused_append_of_tokens_that_are_there_changes_nothing(names):
    c = make()
    a = c.add()
    s = put(c, [a], [range(10)])
    c.fork(a)
    with pytest.raises(ValueError, match="shares the pages"):
        c.append(s, rows(10), rows(10))
    assert c.attend(s, q(), 1.0) == "o"
    c.keep([a], [[2, 4, 6]])
    with pytest.raises(ValueError, match="moved"):
        c.append(s, rows(10), rows(10))
    assert held(names, c, a) == [2, 4, 6] and c.attend(c.step([a], [0]), q(), 1.0) == "o"


def test_a_dropped_sequence_writes_into_no_page(names):
    c = make()
    a = c.add()
    put(c, [a], [range(10)])
    s, done = c.step([a], [3]), c.step([a], [0])
    b = c.fork(a, 10)
    c.drop(a)
    put(c, [b], [[11, 12, 13]])  # in the page that b now holds alone
    for call in (lambda: c.append(s, rows(3), rows(3)), lambda: c.attend(s, q(), 1.0), lambda: c.attend(done, q(), 1.0)):
        with pytest.raises(ValueError, match="dropped"):
            call()
    assert held(names, c, b) == list(range(10)) + [11, 12, 13]


def test_a_step_with_a_dropped_sequence_among_others(names):
    c = make()
    a, b = c.add(), c.add()
    put(c, [a, b], [range(20), range(30)])
    both, one = c.step([a, b], [1, 2]), c.step([a, b], [0, 1])
    c.drop(a)
    with pytest.raises(ValueError, match="dropped"):
        c.append(both, rows(3), rows(3), packed=True)
    with pytest.raises(ValueError, match="not appended"):  # b lacks its tokens of that step
        c.attend(c.step([b], [0]), q(), 1.0)
    c.append(one, rows(1), rows(1), packed=True)  # no new tokens of a
    for step in (both, one):  # a's pages may be another's
        with pytest.raises(ValueError, match="dropped"):
            c.attend(step, q(2), 1.0)
    whole(c)


def test_a_dropped_sequence_and_a_pool_of_another_size(names):
    c = make()
    a, b = c.add(), c.add()
    s = c.step([a], [40])
    put(c, [b], [range(40)])
    c.drop(a)
    c.resize(4)  # b's pages now have the ids that a's step names
    with pytest.raises(ValueError):
        c.append(s, rows(40), rows(40))
    assert held(names, c, b) == list(range(40))


def test_only_the_steps_that_reach_what_moved_are_refused(names):
    c = make()
    a = c.add()
    early = put(c, [a], [range(16)])
    late = put(c, [a], [range(16, 40)])
    c.fork(a)
    put(c, [a], [[40]])  # the third page is copied for a
    assert c.attend(early, q(), 1.0) == "o"
    with pytest.raises(ValueError, match="moved"):
        c.attend(late, q(), 1.0)
    c.keep([a], [list(range(20)) + [30]])
    assert c.attend(early, q(), 1.0) == "o"  # the first page stayed where it was
    c.resize(12)
    with pytest.raises(ValueError, match="moved"):
        c.attend(early, q(), 1.0)


def test_a_step_cut_away_writes_into_no_page(names):
    c = make()
    a, b = c.add(), c.add()
    s = c.step([a], [20])
    c.trim(a, 0)
    put(c, [b], [range(20)])  # in the pages that a's step names
    for call in (lambda: c.append(s, rows(20), rows(20)), lambda: c.attend(s, q(), 1.0)):
        with pytest.raises(ValueError, match="cut"):
            call()
    assert held(names, c, b) == list(range(20))
    assert c.attend(put(c, [a], [[1, 2]]), q(), 1.0) == "o"  # nothing of the refused step is left


def test_a_step_cut_in_the_middle_before_its_append(names):
    c = make()
    a, b = c.add(), c.add()
    s = c.step([a], [40])
    c.trim(a, 20)
    put(c, [b], [range(20)])
    with pytest.raises(ValueError, match="cut"):
        c.append(s, rows(40), rows(40))
    assert held(names, c, b) == list(range(20))
    with pytest.raises(ValueError, match="not appended"):
        c.attend(c.step([a], [0]), q(), 1.0)
    c.trim(a, 0)
    assert c.attend(put(c, [a], [range(3)]), q(), 1.0) == "o"


def test_cut_and_grown_again(names):
    """The length alone does not tell: the tokens are another step's."""
    c = make()
    a = c.add()
    early, s = put(c, [a], [range(10)]), c.step([a], [30])
    c.trim(a, 10)
    now = put(c, [a], [range(100, 130)])
    with pytest.raises(ValueError, match="cut"):
        c.append(s, rows(30), rows(30))
    assert held(names, c, a) == list(range(10)) + list(range(100, 130))
    assert c.attend(early, q(), 1.0) == c.attend(now, q(), 1.0) == "o"
    c.trim(a, 40)  # nothing is forgotten
    assert c.attend(now, q(), 1.0) == "o"


def test_kept_prefixes_cut_the_steps_behind_them(names):
    c = make()
    a, b = c.add(), c.add()
    s, early = put(c, [a], [range(40)]), c.step([a], [0])
    c.keep([a], [range(16)])  # nothing moves
    put(c, [b], [range(24)])
    for step in (s, early):
        with pytest.raises(ValueError, match="cut"):
            c.attend(step, q(), 1.0)
    c.drop(a)
    whole(c)


def test_drafts_round_by_round(names):
    """A step of drafts, its attention, the rejected ones trimmed: the steps of later rounds are as before."""
    c = make()
    a, b = c.add(), c.add()
    put(c, [a, b], [range(30), range(5)])
    want = {a: list(range(30)), b: list(range(5))}
    for i in range(12):
        drafts = {h: [1000 * (h + 1) + 10 * i + j for j in range(4)] for h in (a, b)}
        s = put(c, [a, b], [drafts[a], drafts[b]])
        assert c.attend(s, q(2), 1.0) == "o"
        for h, n in ((a, i % 5), (b, (i + 2) % 5)):
            want[h] += drafts[h][:n]
            c.trim(h, len(want[h]))
            assert held(names, c, h) == want[h]
    whole(c)
    assert len(c._uses) <= 1  # only steps that someone holds


def test_a_refused_step_overtakes_nothing(names):
    c = make()
    a = c.add()
    s = put(c, [a], [range(20)])
    c.fork(a)
    names["fail"] = "copy"
    with pytest.raises(ValueError, match="refused"):
        c.step([a], [1])
    assert c.attend(s, q(), 1.0) == "o"  # its pages are where they were
    c.step([a], [1])
    with pytest.raises(ValueError, match="moved"):
        c.attend(s, q(), 1.0)


def test_an_append_again_that_was_refused(names):
    """attend refuses the sequence until it is put right, and nothing copies or moves what it refuses to read."""
    c = make()
    a = c.add()
    put(c, [a], [range(10)])
    s = put(c, [a], [range(10, 13)])
    with pytest.raises(ValueError, match="different counts"):
        c.append(s, rows(4), rows(4))
    for call in (lambda: c.attend(s, q(), 1.0), lambda: c.fork(a), lambda: c.keep([a], [[1, 11]]), lambda: c.resize(20)):
        with pytest.raises(ValueError, match="not appended"):
            call()
    assert held(names, c, c.fork(a, 10)) == list(range(10))
    c.trim(a, 10)
    assert c.attend(put(c, [a], [[5]]), q(), 1.0) == "o"
    c.resize(20)
    c.keep([a], [[1, 10]])
    assert held(names, c, a) == [1, 5] and c.attend(c.step([a], [0]), q(), 1.0) == "o"


@pytest.mark.parametrize("seed", range(12))
def test_old_steps_in_any_order(names, monkeypatch, seed):
    """Random calls with steps held from before: an append is refused or writes its sequences' own tokens and no others, an attend
    is refused or finds, where its step's table says, the tokens that its sequences have there now."""
    rng = random.Random(seed)
    c, fresh = make(20), iter(range(10 ** 6))
    want, steps, accepted = {c.add(): []}, [], {"append": 0, "attend": 0}
    monkeypatch.setattr(kv8.ops, "kv8_attend_packed", lambda q, pages, scales, table, *a: table)
    lacking = {}  # handle -> positions reserved and never appended

    def step(hs, counts):
        s = c.step(hs, counts)
        for h, n in zip(hs, counts):
            at = len(want[h])
            lacking.setdefault(h, set()).update(range(at, at + n))
            want[h] += [None] * n
        steps.append(s)
        del steps[:-8]
        return s

    def append(s):
        new = [[next(fresh) for _ in range(n)] for _, _, n in s.spans]
        flat = [x for t in new for x in t]
        k = torch.tensor(flat, dtype=torch.float64).view(1, 1, -1, 1).expand(1, HK, len(flat), D)
        try:
            c.append(s, k, k, packed=True)
        except ValueError:
            return
        accepted["append"] += 1
        for (h, at, n), t in zip(s.spans, new):
            if n:
                want[h][at:at + n] = t
                lacking[h].difference_update(range(at, at + n))

    def attend(s):
        try:
            table = c.attend(s, torch.zeros(1, 4, sum(s.counts), D), 1.0, packed=True)
        except ValueError:
            return
        accepted["attend"] += 1
        at = names["pools"].get(c.pages.data_ptr(), {})
        for b, (h, first, n) in enumerate(s.spans):
            for p in range(first + n):
                if p not in lacking.get(h, ()):
                    assert at[int(table[b, p // PAGE])][p % PAGE] == want[h][p]

    for _ in range(400):
        what = rng.choice(["add", "fork", "step", "step", "append", "append", "put", "attend", "attend", "trim", "keep", "drop", "resize"])
        h = rng.choice(list(want)) if want else None
        try:
            if what == "add" or h is None:
                want[c.add()] = []
            elif what == "fork":
                n = rng.randint(0, len(want[h]))
                want[c.fork(h, n)] = list(want[h][:n])
            elif what in ("step", "put"):
                hs = rng.sample(list(want), rng.randint(1, min(3, len(want))))
                s = step(hs, [rng.choice([0, 1, 3, 20]) for _ in hs])
                if what == "put":
                    append(s)
            elif what in ("append", "attend"):
                if steps:
                    (append if what == "append" else attend)(rng.choice(steps))
            elif what == "trim":
                n = rng.randint(0, len(want[h]))
                c.trim(h, n)
                del want[h][n:]
                lacking[h] = {p for p in lacking.get(h, ()) if p < n}
            elif what == "keep":
                at = sorted(rng.sample(range(len(want[h])), rng.randint(0, len(want[h]))))
                c.keep([h], [at])
                want[h] = [want[h][i] for i in at]
                lacking[h] = set()
            elif what == "drop":
                c.drop(h)
                del want[h]
                lacking.pop(h, None)
            else:
                c.resize(rng.randint(14, 24))
        except ValueError as e:
            assert any(x in str(e) for x in ("free", "fit", "not appended")), e
        whole(c)
        at = names["pools"].get(c.pages.data_ptr(), {})
        for x, t in want.items():
            ids = c._seqs[x][0]
            for p, v in enumerate(t):
                if p not in lacking.get(x, ()):
                    assert at[ids[p // PAGE]][p % PAGE] == v
    assert accepted["append"] > 20 and accepted["attend"] > 5
