"""Workspaces of the calls: a captured graph keeps what it captured whatever is called afterwards, and threads that
share a stream keep apart.

Outputs are compared with the same call's made alone, bit for bit: the kernels' results do not depend on what runs beside."""
import threading

import pytest
import torch

from larder_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def cache(B, n, hk=2, d=128, page=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    per = -(-n // page)
    pages = (torch.randn(B * per, 2, hk, page, d, generator=g) * 40).cuda().to(torch.float8_e4m3fn)
    table = torch.randperm(B * per, generator=g).view(B, per).to(torch.int32).cuda()
    return pages, torch.full((B * per, 2, hk), 0.02, device="cuda"), table, i32([n - 7 * b for b in range(B)])


def attend(B, n, seed=0):
    c = cache(B, n, seed=seed)
    q = torch.randn(B, 8, 1, 128, generator=torch.Generator().manual_seed(seed + 1)).to(BF).cuda()
    return lambda: ops.kv8_attend(q, *c, 0.1)


def packed(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(1, sum(lens), h, 128, generator=g).to(BF).cuda().transpose(1, 2) for h in (8, 2, 2))
    cu = i32([sum(lens[:i]) for i in range(len(lens) + 1)])
    return lambda: ops.attn_packed(q, k, v, 0.1, cu)


def decode(B, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, h, t, 128, generator=g).to(BF).cuda() for h, t in ((8, 1), (2, n), (2, n)))
    lens = i32([n - 11 * b for b in range(B)])
    return lambda: ops.attn_decode(q, k, v, 0.1, kv_len=lens)


def partial(B, n):
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(B, h, t, 128, generator=g).to(BF).cuda() for h, t in ((8, 1), (2, n), (2, n)))
    return lambda: ops.attn_decode_partial(q, k, v, 0.1)[0]


def tiled(T, N):
    g = torch.Generator().manual_seed(N)
    q, k, v = (torch.randn(1, h, t, 128, generator=g).to(BF).cuda() for h, t in ((4, T), (2, N), (2, N)))
    m = (torch.rand(T, N, generator=g) < 0.3).cuda()
    m[:, 64:512] = False
    return lambda: ops.attn_prefill_tiled(q, k, v, 0.1, m)


def gdn(T):
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(1, T, 2, 128, generator=g).to(BF).cuda() * 0.1 for _ in range(3))
    a, b = torch.rand(1, T, 2, generator=g).cuda(), torch.rand(1, T, 2, generator=g).cuda()
    return lambda: ops.gdn_chunked(q, k, v, a, b)[0]


def replay_after(small, large):
    """small captured; large called eagerly on the same stream; memory taken and filled; small replayed."""
    want = small().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        small()
    s.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        o = small()
    with torch.cuda.stream(s):
        large()
        held = [torch.full((1 << k,), 7, dtype=torch.uint8, device="cuda") for k in range(9, 24) for _ in range(8)]
        o.zero_()
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want)
    assert all(bool((h == 7).all()) for h in held)
    assert ops.status() == 0


def test_replay_after_a_larger_attention():
    replay_after(attend(2, 500), attend(24, 3000))


def test_replay_after_more_prompts():
    replay_after(packed([40, 300]), packed([30] * 2500))


@pytest.mark.parametrize("make,small,large", [(decode, (2, 500), (24, 6000)), (partial, (1, 900), (16, 5000)),
                                              (tiled, (200, 700), (1500, 4000)), (gdn, (100,), (3000,))])
def test_replay_after_a_larger_call(make, small, large):
    replay_after(make(*small), make(*large))


def test_threads_on_one_stream():
    calls = [decode(2, 600 + 150 * i, seed=i) for i in range(3)]
    calls += [attend(3, 700 + 100 * i, seed=i) for i in range(4)] + [packed([50 + 90 * i, 20, 333], seed=i) for i in range(4)]
    want = [f().clone() for f in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]

    def work(i):
        for _ in range(60):
            got[i].append(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(g) == 60 for g in got)
    assert all(torch.equal(o, w) for g, w in zip(got, want) for o in g)
    assert ops.status() == 0
