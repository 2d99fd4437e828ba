"""kv8.Cache on the host, steps that what happened since has overtaken: which appends and attends are refused, and that none of
them reaches pages or tokens that are not the step's."""
import pytest
import torch

from test_kv8_shared_cpu import D, HK, held, make, names, put, whole  # noqa: F401 (names: the kernels' stand-ins)


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
