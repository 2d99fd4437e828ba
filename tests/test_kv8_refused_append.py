"""kv8.Cache after a refused append, on the host: the step's tokens count, the pages do not hold them, so attention over them
is refused until they are appended or forgotten. The kernels' calls are stood in for."""
import pytest
import torch

from larder_b200 import kv8


@pytest.fixture
def calls(monkeypatch):
    """What reaches the kernels; `fail` makes the next append be refused there."""
    seen = {"append": 0, "attend": 0, "fail": False}

    def append(*a, **kw):
        if seen["fail"]:
            seen["fail"] = False
            raise ValueError("kv8_append: refused")
        seen["append"] += 1

    def attend(*a):
        seen["attend"] += 1
        return "o"

    monkeypatch.setattr(kv8.ops, "kv8_append", append)
    monkeypatch.setattr(kv8.ops, "kv8_attend", attend)
    return seen


def rows(B, T, hk=2, d=64):
    return torch.zeros(B, hk, T, d)


def make():
    c = kv8.Cache(16, 16, 2, 64, device="cpu")
    return c, c.add(), c.add()


def test_refused_by_the_cache_or_the_kernel(calls):
    c, a, b = make()
    step = c.step([a, b], [5, 5])
    for bad in (lambda: c.append(step, rows(2, 4), rows(2, 4)), lambda: c.append(step, rows(1, 9), rows(1, 9), packed=True)):
        with pytest.raises(ValueError):
            bad()
        with pytest.raises(ValueError, match="not appended"):
            c.attend(step, rows(2, 5, 4), 1.0)
    calls["fail"] = True
    with pytest.raises(ValueError, match="refused"):
        c.append(step, rows(2, 5), rows(2, 5))
    with pytest.raises(ValueError, match="not appended"):
        c.attend(step, rows(2, 5, 4), 1.0)
    none = c.step([a, b], [0, 0])
    c.append(none, rows(2, 0), rows(2, 0))  # no tokens: nothing found
    with pytest.raises(ValueError, match="not appended"):
        c.attend(none, rows(2, 1, 4), 1.0)
    assert calls["attend"] == 0
    c.append(step, rows(2, 5), rows(2, 5))  # the same step again, as it should be
    assert c.attend(step, rows(2, 5, 4), 1.0) == "o" and c.length(a) == 5


def test_later_steps_and_other_sequences(calls):
    c, a, b = make()
    first = c.step([a, b], [3, 3])
    c.append(first, rows(2, 3), rows(2, 3))
    bad = c.step([a], [2])
    with pytest.raises(ValueError):
        c.append(bad, rows(1, 1), rows(1, 1))
    assert c.attend(first, rows(2, 3, 4), 1.0) == "o"  # what came before the refused tokens
    only = c.step([b], [1])
    c.append(only, rows(1, 1), rows(1, 1))
    assert c.attend(only, rows(1, 1, 4), 1.0) == "o"  # another sequence
    later = c.step([a, b], [1, 1])
    c.append(later, rows(2, 1), rows(2, 1))
    with pytest.raises(ValueError, match="not appended"):  # over them, two steps on
        c.attend(later, rows(2, 1, 4), 1.0)
    c.trim(a, 3)  # forgotten
    again = c.step([a, b], [1, 1])
    c.append(again, rows(2, 1), rows(2, 1))
    assert c.attend(again, rows(2, 1, 4), 1.0) == "o"


def test_a_new_step_in_their_place_or_a_dropped_sequence(calls):
    c, a, b = make()
    bad = c.step([a, b], [4, 4])
    with pytest.raises(ValueError):
        c.append(bad, rows(2, 1), rows(2, 1))
    c.trim(a, 2)  # in the middle: the first two are still missing
    half = c.step([a], [1])
    c.append(half, rows(1, 1), rows(1, 1))
    with pytest.raises(ValueError, match="not appended"):
        c.attend(half, rows(1, 1, 4), 1.0)
    c.trim(a, 0)
    whole = c.step([a], [4])
    c.append(whole, rows(1, 4), rows(1, 4))
    assert c.attend(whole, rows(1, 4, 4), 1.0) == "o"
    c.drop(b)
    n = c.add()
    step = c.step([n], [7])
    c.append(step, rows(1, 7), rows(1, 7))
    assert c.attend(step, rows(1, 7, 4), 1.0) == "o"
