"""Causal attention over packed prompts on the GPU against 64-bit softmax attention prompt by prompt.

Tolerance: the weights are rounded to the 16-bit type before the second product (relative u), scores are fp32 sums of D
products (under u again for these sizes), the result is rounded once (u): |err| <= u |o| + 2 u sum p |v|. fp32: the
exact kernel, sums of at most 1500 terms: 1e-4 sum p |v|."""
import pytest
import torch

from larder_b200 import ops

import serve_ref as ref

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def cu_of(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()


def inputs(lens, Hq, Hkv, D, dtype, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + pad
    return [torch.randn(1, T, h, D, generator=g).to(dtype).cuda().transpose(1, 2) for h in (Hq, Hkv, Hkv)]


def check(o, q, k, v, lens, scale):
    G, u = q.shape[1] // k.shape[1], ref.UNIT[q.dtype]
    at = 0
    for n in lens:
        for h in range(q.shape[1]):
            a = slice(at, at + n)
            s = (q[0, h, a].double() @ k[0, h // G, a].double().T * scale)
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), -float("inf"))
            p = torch.softmax(s, -1)
            vv = v[0, h // G, a].double()
            want, mass = p @ vv, p @ vv.abs()
            tol = u * want.abs() + (1e-4 if q.dtype == F else 2 * u) * mass
            err = (o[0, h, a].double() - want).abs()
            assert (err <= tol).all(), (n, h, (err / tol).max())
        at += n
    assert ops.status() == 0


LENS = [[1], [5, 1, 3], [128], [129, 127], [256, 256], [257], [0, 40, 0, 0, 300, 0], [700, 1, 64, 63, 65, 513], [1500]]


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 4), (128, 8, 2), (256, 6, 2), (128, 7, 1), (64, 65, 1), (256, 16, 1)])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_packed(dtype, D, Hq, Hkv, lens):
    q, k, v = inputs(lens, Hq, Hkv, D, dtype)
    o = ops.attn_packed(q, k, v, D ** -0.5, cu_of(lens))
    check(o, q, k, v, lens, D ** -0.5)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_prompts(D):
    lens = [(i * 37) % 61 for i in range(200)]
    q, k, v = inputs(lens, 2, 1, D, BF)
    check(ops.attn_packed(q, k, v, 0.3, cu_of(lens)), q, k, v, lens, 0.3)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 2, 1), (256, 2, 1), (256, 3, 3)])
def test_long_prompts(D, Hq, Hkv, dtype):
    """Prompts long enough on average for every form of the kernels, short ones among them."""
    lens = [4001, 7, 0, 9000, 130]
    q, k, v = inputs(lens, Hq, Hkv, D, dtype)
    check(ops.attn_packed(q, k, v, D ** -0.5, cu_of(lens)), q, k, v, lens, D ** -0.5)
    lens = [6500, 0, 200, 5400]
    q, k, v = inputs(lens, Hq, Hkv, D, dtype, seed=1, pad=300)
    out = torch.full_like(q, 9.0)
    check(ops.attn_packed(q, k, v, D ** -0.5, cu_of(lens), out=out), q, k, v, lens, D ** -0.5)
    assert (out[:, :, 12100:] == 0).all()
    v[0, 0, 6500 + 111, 3] = float("nan")  # reaches the later rows of its own prompt
    o = ops.attn_packed(q, k, v, D ** -0.5, cu_of(lens))
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[0, :Hq // Hkv, 6500 + 111:6700, 3] = True
    assert torch.equal(torch.isnan(o), bad)
    assert ((o - out).abs()[~bad].double() <= 6 * ref.UNIT[dtype] * v.nan_to_num(0).abs().max()).all()


def test_wrong_bounds_stay_inside():
    """Bounds that fall or leave the rows are clamped: nothing outside the tensors is touched, whatever comes out."""
    q, k, v = inputs([300], 4, 2, 128, BF)
    wide = torch.full((1, 310, 4, 128), 5.0, dtype=BF, device="cuda")
    out = wide[:, 5:305].transpose(1, 2)
    for cu in ([0, 200, 100, 300], [-50, 20, 5000], [300, 0], [0, 1 << 30]):
        for f, a in ((BF, (q, k, v)), (F, (q.float(), k.float(), v.float()))):
            o = ops.attn_packed(*a, 0.1, torch.tensor(cu, dtype=torch.int32).cuda(), out=out if f is BF else None)
            torch.cuda.synchronize()
    assert (wide[:, :5] == 5).all() and (wide[:, 305:] == 5).all() and ops.status() == 0


@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_of_no_prompt_are_zero(dtype):
    lens = [100, 30]
    q, k, v = inputs(lens, 4, 2, 128, dtype, pad=75)
    out = torch.full_like(q, 9.0)
    ops.attn_packed(q, k, v, 0.1, cu_of(lens), out=out)
    check(out, q, k, v, lens, 0.1)
    assert (out[:, :, 130:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_unseen_infinities_and_nan(dtype, D):
    """Non-finite keys and values reach the rows that see them and no others: not another prompt's, not an earlier row."""
    lens = [70, 300, 33]
    q, k, v = inputs(lens, 4, 2, D, dtype, seed=2)
    clean = ops.attn_packed(q, k, v, D ** -0.5, cu_of(lens))
    v[0, 0, 70 + 211, 3] = float("nan")
    v[0, 1, 70, 5] = float("inf")
    k[0, 1, 69, 0] = float("nan")     # the first prompt's last key
    k[0, 0, 370 + 10, 1] = float("inf")
    o = ops.attn_packed(q, k, v, D ** -0.5, cu_of(lens))
    touched = torch.zeros_like(o, dtype=torch.bool)
    touched[0, :2, 70 + 211:370] = True
    touched[0, 2:, 70:370] = True
    touched[0, 2:, 69] = True
    touched[0, :2, 380:] = True
    u = ref.UNIT[dtype]
    assert torch.isfinite(o[~touched]).all()
    # untouched rows: both sides within the file's tolerance of the same exact result
    assert ((o - clean).abs()[~touched].double() <= 6 * (u if dtype != F else 1e-4) * v.nan_to_num(0, 0, 0).abs().max()).all()
    assert torch.isnan(o[0, :2, 70 + 211:370, 3]).all() and torch.isnan(o[0, 2:, 69]).all()
    assert (~torch.isfinite(o[0, 2:, 70:370, 5])).all()


def test_strides_out_and_large_offsets():
    lens = [33, 150]
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(1, 183, (8 + 2 + 2) * 128, generator=g).to(BF).cuda()  # one projection's rows
    q, k, v = (x.unflatten(-1, (-1, 128)).transpose(1, 2) for x in qkv.split([8 * 128, 256, 256], -1))
    out = torch.empty(1, 183, 8, 128, dtype=BF, device="cuda").transpose(1, 2)
    assert ops.attn_packed(q, k, v, 0.09, cu_of(lens), out=out) is out
    check(out, q, k, v, lens, 0.09)


def test_large_scores():
    """Scores of some hundreds: far outside the range of exp without a running maximum."""
    lens = [90]
    q, k, v = inputs(lens, 2, 2, 128, HF, seed=6)
    check(ops.attn_packed(q * 20, k, v, 1.0, cu_of(lens)), q * 20, k, v, lens, 1.0)


def test_another_stream():
    lens = [300, 20]
    q, k, v = inputs(lens, 8, 2, 128, BF)
    cu = cu_of(lens)
    want = ops.attn_packed(q, k, v, 0.1, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o = ops.attn_packed(q, k, v, 0.1, cu)
    s.synchronize()
    assert torch.equal(o, want)


def test_refused():
    q, k, v = inputs([8], 4, 2, 128, BF)
    cu = cu_of([8])
    f = ops.attn_packed
    assert f(q[:, :, :0], k[:, :, :0], v[:, :, :0], 1.0, cu_of([0])).shape == (1, 4, 0, 128)
    for bad in (lambda: f(q[:, :3], k, v, 1.0, cu), lambda: f(q, k, v[:, :1], 1.0, cu), lambda: f(q, k.half(), v, 1.0, cu),
                lambda: f(q, k, v, 1.0, cu.long()), lambda: f(q, k, v, 1.0, cu[:1]), lambda: f(q[0], k, v, 1.0, cu),
                lambda: f(q[..., :96], k[..., :96], v[..., :96], 1.0, cu), lambda: f(q[:, :, :4], k, v, 1.0, cu),
                lambda: f(q.cpu(), k, v, 1.0, cu), lambda: f(q, k, v, 1.0, cu, out=torch.empty(1, 4, 8, 64, device="cuda")),
                lambda: f(q, k, v, 0.0, cu), lambda: f(q, k, v, -1.0, cu), lambda: f(q, k, v, float("nan"), cu),
                lambda: f(q.transpose(2, 3), k, v, 1.0, cu), lambda: f(q.double(), k.double(), v.double(), 1.0, cu)):
        with pytest.raises(ValueError):
            bad()
