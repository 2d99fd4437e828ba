"""A host thread's first CUDA call may be one of the library's: calls from fresh threads give what the main thread's give."""
import threading

import pytest
import torch

from larder_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def calls():
    g = torch.Generator().manual_seed(0)

    def r(*shape):
        return torch.randn(*shape, generator=g).to(BF).cuda()

    q, k, v = r(1, 8, 1, 128), r(1, 2, 300, 128), r(1, 2, 300, 128)
    qp, kp, vp = r(1, 8, 40, 128), r(1, 2, 40, 128), r(1, 2, 40, 128)
    cu, n = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 25, 40], [200]))
    pages = (torch.randn(20, 2, 2, 16, 128, generator=g) * 40).cuda().to(torch.float8_e4m3fn)
    scales, table = torch.full((20, 2, 2), 0.02, device="cuda"), torch.arange(20, dtype=torch.int32).cuda()[None]
    return {"attn_decode": lambda: ops.attn_decode(q, k, v, 0.1), "attn_prefill": lambda: ops.attn_prefill(qp, k, v, 0.1),
            "attn_packed": lambda: ops.attn_packed(qp, kp, vp, 0.1, cu),
            "kv8_attend": lambda: ops.kv8_attend(q, pages, scales, table, n, 0.1)}


@pytest.mark.parametrize("name", ["attn_decode", "attn_prefill", "attn_packed", "kv8_attend"])
def test_first_call_of_a_thread(name):
    f = calls()[name]
    want = f()
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(f())
        except Exception as e:  # (shown by the assertion below)
            got.append(e)

    for _ in range(3):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert all(torch.is_tensor(o) and torch.equal(o, want) for o in got), got
