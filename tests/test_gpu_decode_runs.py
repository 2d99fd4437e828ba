"""Split-KV decode of sequences far shorter than the cache's capacity: fewer key tiles in the call than CTAs in its grid, which
is sized by the capacity. The workspace holds huge finite partials beforehand, so that a partial read without having been
written by the call shows. Tolerance: the other decode tests' (weights and outputs in 16 bits): u |o| + 2 u sum p |v|."""
import pytest
import torch

from larder_b200 import _lib, ops

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [[512], [1], [64, 0, 65, 130], [0, 8192, 3], [700] * 6], ids=str)
def test_partials_that_no_cta_wrote(lens, D, dtype):
    B, Hq, Hkv, cap, scale = len(lens), 8, 4, 8192, D ** -0.5
    g = torch.Generator().manual_seed(len(lens) + D)
    q = torch.randn(B, Hq, 1, D, generator=g).to(dtype).cuda()
    k, v = (torch.randn(B, Hkv, cap, D, generator=g).to(dtype).cuda() for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    L = _lib.lib()
    nbytes = L.lb2_attn_decode_workspace_size(B, Hq, Hkv, 1, cap, D, 0)
    ws = torch.full((nbytes // 4 + 64,), 1000.0, device="cuda")
    out, part, lse = torch.empty_like(q), torch.empty(B, Hq, 1, D, device="cuda"), torch.empty(B, Hq, 1, device="cuda")
    code, st = ops.dtype_code(q), torch.cuda.current_stream().cuda_stream
    common = (q.data_ptr(), _lib.i64(*q.stride()[:3]), k.data_ptr(), _lib.i64(*k.stride()[:3]), v.data_ptr(),
              _lib.i64(*v.stride()[:3]))
    for _ in range(2):
        assert L.lb2_attn_decode(*common, out.data_ptr(), _lib.i64(*out.stride()[:3]), n.data_ptr(), B, Hq, Hkv, 1, cap, D,
                                 code, scale, 0, 0, ws.data_ptr(), ws.numel() * 4, st) == 0
        ws.fill_(1000.0)
    assert L.lb2_attn_decode_partial(*common, part.data_ptr(), lse.data_ptr(), n.data_ptr(), B, Hq, Hkv, 1, cap, D, code,
                                     scale, 0, ws.data_ptr(), ws.numel() * 4, st) == 0
    u = ref.UNIT[dtype]
    for b in range(B):
        for h in range(Hq):
            want, mass = ref.attend(q[b, h], k[b, h // 2], v[b, h // 2], scale, [lens[b]])
            for got in (out, part):
                assert ((got[b, h].double() - want).abs() <= u * want.abs() + 2 * u * mass).all(), (b, h)
            if lens[b]:
                s = torch.logsumexp(k[b, h // 2, :lens[b]].double() @ q[b, h, 0].double() * scale, 0)
                assert abs(float(lse[b, h]) - float(s)) <= 1e-3
    assert ops.status() == 0
