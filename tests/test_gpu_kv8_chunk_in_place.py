"""kv8_attend_packed reads rows of q a second time where a NaN code may have reached them, after their results are written: an out
that is q itself is refused, one that lies beside it in the same memory is not."""
import pytest
import torch

from larder_b200 import ops

from test_gpu_kv8_chunk import BF, F, cache, close, expect, i32, queries, starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F])
def test_out_may_not_be_q(dtype):
    lens, counts, d = [300, 260], [140, 100], 128
    pages, scales, table = cache(lens, 1, 16, d)
    both = torch.empty(sum(counts), 4, d, dtype=dtype, device="cuda").transpose(0, 1)[None]  # q's heads, then the result's
    q, out = both[:, :2], both[:, 2:]
    q.copy_(queries(2, sum(counts), d, dtype))
    args = (pages, scales, table, i32(lens), i32(starts(counts)), 0.1)
    o, a = expect(q, pages, scales, table, lens, counts, 0.1)
    pages.view(torch.uint8)[int(table[0, 200 // 16]), 1, 0, 200 % 16, 5] = 0x7F  # a value of sequence 0's new token 40
    for same in (q, q[:, :, :], q.as_strided(q.shape, q.stride())):
        with pytest.raises(ValueError, match="must not be q"):
            ops.kv8_attend_packed(q, *args, out=same)
    ops.kv8_attend_packed(q, *args, out=out)
    assert ops.status() == 0 and torch.isnan(out[0, :, 40:140, 5]).all()
    rest = torch.ones_like(o, dtype=torch.bool)
    rest[:, 40:140, 5] = False
    close(out.masked_fill(~rest, 0), o.masked_fill(~rest, 0), a, dtype)
    none = q[:, :, :0]
    assert ops.kv8_attend_packed(none, pages, scales, table, i32(lens), i32([0, 0, 0]), 0.1, out=none) is none
