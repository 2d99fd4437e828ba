"""Compaction of tokens that hold only zeros in a page of ordinary scale together with tokens of hardly any magnitude: zeros stay
zeros, though the one scale over the other passes fp32's range."""
import pytest
import torch

from larder_b200 import ops
from larder_b200.rope import Rope

from test_gpu_kv8_pages import run_compact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,layout", [(0, "half"), (64, "half"), (64, "interleaved"), (32, "half"), (10, "half")])
@pytest.mark.parametrize("page,d", [(16, 64), (64, 128), (128, 256)])
@pytest.mark.parametrize("small", [2.0 ** -126, 2.0 ** -122])
def test_zeros_of_a_loud_page_among_quiet_tokens(page, d, small, R, layout):
    zero, nan = 3, 5

    def edit(pages, scales, table):
        raw = pages.view(torch.uint8)
        loud, quiet = int(table[0, 0]), int(table[0, 1])
        scales[loud] = 4.0
        raw[loud, :, :, zero] = 0
        raw[loud, :, :, zero, ::3] = 0x80  # (-0)
        raw[loud, :, :, nan] = 0
        raw[loud, :, :, nan, 1] = 0x7F
        scales[quiet] = small

    keep = [zero, nan] + list(range(page, 2 * page - 2))
    pages, scales, table, to = run_compact([2 * page], [keep], [0], 2, page, d, Rope(R, layout=layout) if R else None, edit=edit)
    raw = pages.view(torch.uint8)[int(to[0, 0])]
    assert ((raw[:, :, 0] & 0x7F) == 0).all()
    assert ((raw[1, :, 1] & 0x7F) == 0).sum() == 2 * (d - 1) and ops.status() == 0
