"""The serving example runs: prompts packed, decode steps over the paged 8-bit cache, a sequence replaced. e4m3 keeps 4
significant bits: each key and value is off by 2^-4 of itself at most, so an output is off by less than a tenth of its
norm through the values (whose errors average over the keys) and the keys together."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.gpu
def test_serve_paged():
    import serve_paged
    assert serve_paged.main(steps=4, hidden=512, hq=8, hk=2, d=64, lens=(70, 150, 3, 33)) < 0.1
