"""torch-facing wrappers of the C-ABI entry points: shape/dtype/stride checks, output and workspace allocation,
the caller's current CUDA stream. Every function here runs a CUDA kernel of liblarder_b200; none has a CPU path.

Tensors follow the reference's layouts (mlx_lm's): attention q [B, Hq, T, D] (often a transposed view of
[B, T, Hq, D]), k / v [B, Hkv, N, D] (often slices of a capacity-padded cache buffer); Gated-DeltaNet q / k
[B, T, Hk, Dk], v [B, T, Hv, Dv], state [B, Hv, Dv, Dk] fp32.
"""
import ctypes

import torch

from . import _lib
from ._lib import check, i64, lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_WS = {}  # (device index, tag) -> uint8 workspace, grown on demand


def dtype_code(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}") from None


def _cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("larder_b200 runs on CUDA tensors only (no CPU path)")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t):
    """The caller's current CUDA stream on t's device, as the cudaStream_t handle (an int) the C ABI takes."""
    if _raw_stream is not None:
        return _raw_stream(t.device.index)
    return torch.cuda.current_stream(t.device).cuda_stream


def _stream_of(dev):
    """The same for a device index."""
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


# Scratch of one call, from the caching allocator and given back as soon as the call's kernels are queued: whoever gets the
# memory next on the stream comes after them. Nothing holds its address for a later call, so that a captured graph owns
# what it captured and calls of several threads or streams may run at once. (Addresses, not tensors: 0.5 us against 1.5.)
_scratch = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_alloc", None)
_scratch_done = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_delete", None)
if _scratch is None or _scratch_done is None:
    def _scratch(nbytes, stream):
        return torch.cuda.caching_allocator_alloc(nbytes, stream=stream)

    def _scratch_done(ptr):
        torch.cuda.caching_allocator_delete(ptr)


def _ptr(t):
    """A tensor's device address as the C ABI's void* (None for NULL); the argtypes convert plain ints."""
    return None if t is None else t.data_ptr()


def _unit_last(t, name):
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: the last axis must have unit stride")


def workspace(device, nbytes, tag):
    """A 256-byte aligned uint8 buffer of at least nbytes on device, kept per (device, tag): for attn_decode_host, whose
    staging slots outlive a call, and which waits for the copies in flight before it takes a larger one."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), tag)
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        buf = torch.zeros(max(int(nbytes), 256) + 256, dtype=torch.uint8, device=device)
        ws = buf[(-buf.data_ptr()) % 256:]
        _WS[key] = ws
    return ws


def status(device=None):
    """Synchronise the current stream and return (and clear) the library's device status word (0 = ok)."""
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
    return lib().lb2_status(ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream))


# ---------------------------------------------------------------------------------------------------- attention

def attn_prefill(q, k, v, scale, mask=None, gate=None, out=None):
    """softmax(scale q k^T + mask) v [* sigmoid(gate)] on tcgen05 tensor cores.

    mask: None, "causal" (bottom-right) or a bool tensor broadcastable from [T, N] (leading dims of 1)."""
    _cuda(q, k, v, gate)
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _unit_last(t, n)
    B, Hq, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share a dtype")
    if v.shape[-1] != D:
        raise ValueError("v's head dim must equal q's")
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=q.device)
    kind, m, mst = _lib.MASK_NONE, None, i64(0, 0)
    if isinstance(mask, str):
        if mask != "causal":
            raise ValueError(f"unsupported mask {mask!r}")
        kind = _lib.MASK_CAUSAL
    elif mask is not None:
        if mask.dtype != torch.bool or tuple(mask.shape[-2:]) != (T, N) or any(d != 1 for d in mask.shape[:-2]):
            raise ValueError("array masks must be bool [..., T, N] with leading dims of 1")
        m = mask.reshape(T, N).view(torch.uint8)  # (bool and uint8 share a byte layout: no copy, strides kept)
        kind, mst = _lib.MASK_ARRAY, i64(m.stride(0), m.stride(1))
    gst = i64(0, 0, 0)
    if gate is not None:
        if gate.shape != (B, Hq, T, D) or gate.dtype != q.dtype:
            raise ValueError("gate must be [B, Hq, T, D] in q's dtype")
        _unit_last(gate, "gate")
        gst = i64(*gate.stride()[:3])
    rc = lib().lb2_attn_prefill(_ptr(q), i64(*q.stride()[:3]), _ptr(k), i64(*k.stride()[:3]), _ptr(v),
                                i64(*v.stride()[:3]), _ptr(out), i64(*out.stride()[:3]), _ptr(gate), gst,
                                _ptr(m), mst, B, Hq, Hkv, T, N, D, dtype_code(q), float(scale), kind, _stream(q))
    check(rc, "attn_prefill")
    return out


def attn_prefill_tiled(q, k, v, scale, mask, gate=None, out=None):
    """attn_prefill with a bool array mask [..., T, N] and tile skipping: only the key tiles that some row of a row
    block keeps are read and multiplied (lb2_attn_prefill_tiled). Same result as attn_prefill(..., mask)."""
    _cuda(q, k, v, gate, mask)
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _unit_last(t, n)
    B, Hq, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share a dtype")
    if mask.dtype != torch.bool or tuple(mask.shape[-2:]) != (T, N) or any(d != 1 for d in mask.shape[:-2]):
        raise ValueError("array masks must be bool [..., T, N] with leading dims of 1")
    m = mask.reshape(T, N).view(torch.uint8)  # (no copy, strides kept)
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=q.device)
    gst = i64(0, 0, 0)
    if gate is not None:
        if gate.shape != (B, Hq, T, D) or gate.dtype != q.dtype:
            raise ValueError("gate must be [B, Hq, T, D] in q's dtype")
        _unit_last(gate, "gate")
        gst = i64(*gate.stride()[:3])
    n = lib().lb2_attn_prefill_tiled_workspace_size(T, N, D)
    stream = _stream(q)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_attn_prefill_tiled(_ptr(q), i64(*q.stride()[:3]), _ptr(k), i64(*k.stride()[:3]), _ptr(v),
                                          i64(*v.stride()[:3]), _ptr(out), i64(*out.stride()[:3]), _ptr(gate), gst,
                                          _ptr(m), i64(m.stride(0), m.stride(1)), B, Hq, Hkv, T, N, D, dtype_code(q),
                                          float(scale), ws, n, stream)
    finally:
        _scratch_done(ws)
    check(rc, "attn_prefill_tiled")
    return out


def decode_rows_limit(D):
    """Folded rows (G*T) the split-KV decode kernel takes at head dim D."""
    return 16 if D == 256 else 32


_DECODE_WS = {}  # (B, Hq, Hkv, T, N, D, split, device index) -> workspace bytes (the plan depends on the SM count)


def _decode_ws_bytes(B, Hq, Hkv, T, N, D, split, dev):
    key = (B, Hq, Hkv, T, N, D, split, dev)
    n = _DECODE_WS.get(key)
    if n is None:
        n = _DECODE_WS[key] = lib().lb2_attn_decode_workspace_size(B, Hq, Hkv, T, N, D, split)
    return n


def attn_decode(q, k, v, scale, causal=False, kv_len=None, split=0, out=None):
    """Split-KV decode attention: q [B, Hq, T, D] with few rows over k / v [B, Hkv, N, D]; kv_len int32 [B]
    (on the device) gives each sequence's key count, else all N."""
    _cuda(q, k, v, kv_len)
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _unit_last(t, n)
    B, Hq, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=q.device)
    if kv_len is not None and (kv_len.dtype != torch.int32 or kv_len.numel() != B):
        raise ValueError("kv_len must be int32 [B]")
    n = _decode_ws_bytes(B, Hq, Hkv, T, N, D, split, q.device.index)
    stream = _stream(q)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_attn_decode(_ptr(q), i64(*q.stride()[:3]), _ptr(k), i64(*k.stride()[:3]), _ptr(v),
                                   i64(*v.stride()[:3]), _ptr(out), i64(*out.stride()[:3]), _ptr(kv_len), B, Hq, Hkv, T,
                                   N, D, dtype_code(q), float(scale), int(bool(causal)), int(split), ws, n, stream)
    finally:
        _scratch_done(ws)
    check(rc, "attn_decode")
    return out


def attn_decode_host(q_host, k, v, scale, o_host, causal=False, kv_len=None, split=0):
    """attn_decode for q and o in host memory (contiguous CPU tensors [B, Hq, T, D], pinned for the copies to
    overlap): copies q in, decodes on the current stream, copies o out, without waiting. o_host (of this call and
    the ones before) is complete after attn_decode_host_drain() and a synchronisation of the stream."""
    _cuda(k, v, kv_len)
    for t, n in ((q_host, "q_host"), (o_host, "o_host")):
        if t.is_cuda or not t.is_contiguous():
            raise ValueError(f"attn_decode_host: {n} must be a contiguous host tensor")
    if q_host.shape != o_host.shape or q_host.dtype != o_host.dtype or q_host.dtype != k.dtype:
        raise ValueError("attn_decode_host: q_host, o_host and the cache must share shape / dtype")
    B, Hq, T, D = q_host.shape
    Hkv, N = k.shape[1], k.shape[2]
    if kv_len is not None and (kv_len.dtype != torch.int32 or kv_len.numel() != B):
        raise ValueError("kv_len must be int32 [B]")
    L = lib()
    need = L.lb2_attn_decode_host_workspace_size(B, Hq, Hkv, T, N, D, dtype_code(k), int(split))
    cur = _WS.get((k.device.index if k.device.index is not None else torch.cuda.current_device(), "decode_host"))
    if cur is not None and cur.numel() < need:  # copies still in flight may use the old buffer: let them finish
        attn_decode_host_drain(k.device.index)
        torch.cuda.synchronize(k.device)
    ws = workspace(k.device, need, "decode_host")
    rc = L.lb2_attn_decode_host(q_host.data_ptr(), _ptr(k), i64(*k.stride()[:3]), _ptr(v), i64(*v.stride()[:3]),
                                o_host.data_ptr(), _ptr(kv_len), B, Hq, Hkv, T, N, D, dtype_code(k), float(scale),
                                int(bool(causal)), int(split), _ptr(ws), ws.numel(), _stream(k))
    check(rc, "attn_decode_host")
    return o_host


def attn_decode_host_drain(device=None):
    """Order the current stream after every outstanding attn_decode_host copy out."""
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
    check(lib().lb2_attn_decode_host_drain(ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)),
          "attn_decode_host_drain")


def attn_decode_partial(q, k, v, scale, kv_len=None, split=0, out=None):
    """This KV range's normalised partial output (fp32 [B, Hq, T, D]) and log-sum-exp (fp32 [B, Hq, T]); `out`, a
    pair of contiguous fp32 tensors of those shapes (for instance the two parts of one packed exchange buffer),
    receives them when given."""
    _cuda(q, k, v, kv_len)
    B, Hq, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    if out is None:
        part_o = torch.empty((B, Hq, T, D), dtype=torch.float32, device=q.device)
        part_lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device)
    else:
        part_o, part_lse = out
        for t, shp in ((part_o, (B, Hq, T, D)), (part_lse, (B, Hq, T))):
            if t.dtype != torch.float32 or tuple(t.shape) != shp or not t.is_contiguous() or t.device != q.device:
                raise ValueError(f"attn_decode_partial: out must be contiguous fp32 {shp} on q's device")
    decode_partial_into(q, k, v, scale, kv_len, split, _ptr(part_o), _ptr(part_lse))
    return part_o, part_lse


def decode_partial_into(q, k, v, scale, kv_len, split, part_o_ptr, part_lse_ptr):
    """attn_decode_partial into raw device addresses (contiguous fp32 [B, Hq, T, D] and [B, Hq, T]): the halves of
    a peer-exchange buffer, which no tensor wraps."""
    B, Hq, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    n = _decode_ws_bytes(B, Hq, Hkv, T, N, D, split, q.device.index)
    stream = _stream(q)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_attn_decode_partial(_ptr(q), i64(*q.stride()[:3]), _ptr(k), i64(*k.stride()[:3]), _ptr(v),
                                           i64(*v.stride()[:3]), part_o_ptr, part_lse_ptr, _ptr(kv_len), B, Hq, Hkv,
                                           T, N, D, dtype_code(q), float(scale), int(split), ws, n, stream)
    finally:
        _scratch_done(ws)
    check(rc, "attn_decode_partial")


def decode_push(q, k, v, scale, kv_len, split, bufs, R, rank, epoch):
    """This rank's KV-range partial stored into slot `rank` of half epoch % 2 of every rank's push-exchange buffer
    (bufs: a ctypes uint64 array of the R buffers as mapped here), lb2_attn_decode_push."""
    B, Hq, T, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    n = _decode_ws_bytes(B, Hq, Hkv, T, N, D, split, q.device.index)
    stream = _stream(q)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_attn_decode_push(_ptr(q), i64(*q.stride()[:3]), _ptr(k), i64(*k.stride()[:3]), _ptr(v),
                                        i64(*v.stride()[:3]), _ptr(kv_len), B, Hq, Hkv, T, N, D, dtype_code(q),
                                        float(scale), int(split), ws, n, bufs, int(R), int(rank), int(epoch), stream)
    finally:
        _scratch_done(ws)
    check(rc, "attn_decode_push")


def attn_combine(part_o, part_lse, dtype, out=None):
    """Merge R partials part_o [R, B, Hq, T, D], part_lse [R, B, Hq, T] (fp32) by log-sum-exp."""
    _cuda(part_o, part_lse)
    R, B, Hq, T, D = part_o.shape
    part_o, part_lse = part_o.contiguous(), part_lse.contiguous()
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=dtype, device=part_o.device)
    rc = lib().lb2_attn_combine(_ptr(part_o), _ptr(part_lse), R, B, Hq, T, D, _ptr(out), i64(*out.stride()[:3]),
                                dtype_code(out), _stream(part_o))
    check(rc, "attn_combine")
    return out


def attn_combine_packed(gathered, R, B, Hq, T, D, dtype, out=None):
    """Merge R partials from an all-gathered packed buffer: R blocks of [o rows (B Hq T D) | lse (B Hq T)] fp32."""
    _cuda(gathered)
    if gathered.dtype != torch.float32 or not gathered.is_contiguous() or gathered.numel() != R * B * Hq * T * (D + 1):
        raise ValueError("attn_combine_packed: gathered must be contiguous fp32 of R * B * Hq * T * (D + 1) values")
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=dtype, device=gathered.device)
    rc = lib().lb2_attn_combine_packed(_ptr(gathered), R, B, Hq, T, D, _ptr(out), i64(*out.stride()[:3]),
                                       dtype_code(out), _stream(gathered))
    check(rc, "attn_combine_packed")
    return out


# ---------------------------------------------------------------------------------------------------- GDN

def _gdn_common(q, k, v, g, beta, state):
    _cuda(q, k, v, g, beta, state)
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    if k.shape != q.shape or k.dtype != q.dtype:
        raise ValueError("q and k must share shape and dtype")
    if state is None:
        state = torch.zeros((B, Hv, Dv, Dk), dtype=torch.float32, device=q.device)
    if state.dtype != torch.float32 or tuple(state.shape) != (B, Hv, Dv, Dk):
        raise ValueError("state must be fp32 [B, Hv, Dv, Dk]")
    q, k, v, g, beta, state = (t.contiguous() for t in (q, k, v, g, beta, state))
    return q, k, v, g, beta, state, (B, T, Hk, Dk, Hv, Dv)


def gdn_recurrent(q, k, v, g, beta, state=None, mask=None, state_out=None):
    """The gated delta recurrence position by position: returns (y [B, T, Hv, Dv] in q's dtype, new state). The new
    state goes to `state_out` when given (fp32, the state's shape, contiguous, not the input state itself)."""
    q, k, v, g, beta, state, (B, T, Hk, Dk, Hv, Dv) = _gdn_common(q, k, v, g, beta, state)
    y = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=q.device)
    if state_out is None:
        s_out = torch.empty_like(state)
    else:
        if (state_out.shape != state.shape or state_out.dtype != torch.float32 or not state_out.is_contiguous()
                or state_out.data_ptr() == state.data_ptr()):
            raise ValueError("gdn_recurrent: state_out must be a separate contiguous fp32 tensor of the state's shape")
        s_out = state_out
    m = None
    if mask is not None:
        m = mask.reshape(B, T).to(torch.uint8).contiguous()
    rc = lib().lb2_gdn_recurrent(_ptr(q), _ptr(k), dtype_code(q), _ptr(v), dtype_code(v), _ptr(g), dtype_code(g),
                                 int(g.dim() == 4), _ptr(beta), dtype_code(beta), _ptr(m), _ptr(state), _ptr(s_out),
                                 _ptr(y), B, T, Hk, Dk, Hv, Dv, _stream(q))
    check(rc, "gdn_recurrent")
    return y, s_out


def gdn_chunked_supported(q, v, g, mask):
    return (mask is None and g.dim() == 3 and q.shape[-1] == 128 and v.shape[-1] == 128
            and q.dtype in (torch.bfloat16, torch.float16))


def gdn_chunked(q, k, v, g, beta, state=None):
    """The same recurrence in chunks of 64 positions on tensor cores (scalar gate, no mask, Dk = Dv = 128)."""
    q, k, v, g, beta, state, (B, T, Hk, Dk, Hv, Dv) = _gdn_common(q, k, v, g, beta, state)
    y = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=q.device)
    s_out = torch.empty_like(state)
    nbytes = lib().lb2_gdn_chunked_workspace_size(B, T, Hk, Hv, Dk, Dv)
    stream = _stream(q)
    ws = _scratch(nbytes or 1, stream)
    try:
        rc = lib().lb2_gdn_chunked(_ptr(q), _ptr(k), dtype_code(q), _ptr(v), dtype_code(v), _ptr(g), dtype_code(g),
                                   _ptr(beta), dtype_code(beta), _ptr(state), _ptr(s_out), _ptr(y), B, T, Hk, Dk, Hv,
                                   Dv, ws, nbytes, stream)
    finally:
        _scratch_done(ws)
    check(rc, "gdn_chunked")
    return y, s_out


# ---------------------------------------------------------------------------------------------------- gathers

def kv_gather_picks(k, v, tb, cr, n=None):
    """Rows of one sequence's k / v [Hk, n, D] (or [1, Hk, n, D]) that QSA decode attends to: the sorted picked
    blocks tb (int32, block size cr) and the trailing partial block. Returns kg, vg [1, Hk, m, D]."""
    _cuda(k, v, tb)
    if k.dim() == 4:
        k, v = k[0], v[0]
    Hk, N, D = k.shape
    n = N if n is None else int(n)
    tb = tb.reshape(-1)
    if tb.dtype != torch.int32:
        raise ValueError("tb must be int32")
    nsel = tb.numel()
    m = nsel * cr + n - n // cr * cr
    kg = torch.empty((1, Hk, m, D), dtype=k.dtype, device=k.device)
    vg = torch.empty_like(kg)
    rc = lib().lb2_kv_gather_picks(_ptr(k), i64(*k.stride()), _ptr(v), i64(*v.stride()), _ptr(tb), nsel, int(cr), n,
                                   _ptr(kg), _ptr(vg), Hk, D, dtype_code(k), _stream(k))
    check(rc, "kv_gather_picks")
    return kg, vg


def qsa_decode(q, k, v, tb, cr, scale, n=None, out=None):
    """One QSA decode row with the gather inside the decode kernel: q [1, Hq, 1, D] attends to the rows of k / v
    [Hk, n, D] (or [1, Hk, n, D]) that kv_gather_picks(k, v, tb, cr) would return, read in place. Bit-equal to
    attn_decode over kv_gather_picks' output."""
    _cuda(q, k, v, tb)
    if k.dim() == 4:
        k, v = k[0], v[0]
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        _unit_last(t, nm)
    Hk, N, D = k.shape
    n = N if n is None else int(n)
    tb = tb.reshape(-1)
    if tb.dtype != torch.int32:
        raise ValueError("tb must be int32")
    _, Hq, T, _ = q.shape
    if q.shape[0] != 1 or T != 1:
        raise ValueError("qsa_decode: one query row [1, Hq, 1, D]")
    if out is None:
        out = torch.empty_like(q)
    nsel = tb.numel()
    L = lib()
    nbytes = L.lb2_qsa_decode_workspace_size(nsel, int(cr), n, Hq, Hk, D)
    stream = _stream(q)
    ws = _scratch(nbytes or 1, stream)
    try:  # (the views as [1, Hk, n, D]: a batch stride of Hk heads, for the tensor maps the kernel is given)
        rc = L.lb2_qsa_decode(_ptr(q), i64(*q.stride()[:3]), _ptr(k), i64(Hk * k.stride(0), *k.stride()[:2]), _ptr(v),
                              i64(Hk * v.stride(0), *v.stride()[:2]), _ptr(out), i64(*out.stride()[:3]), _ptr(tb), nsel,
                              int(cr), n, Hq, Hk, D, dtype_code(q), float(scale), ws, nbytes, stream)
    finally:
        _scratch_done(ws)
    check(rc, "qsa_decode")
    return out


def kvh_put(table, k, v, pos0, logc):
    """Write k / v [Hk, s, D] (or [1, Hk, s, D]) as positions pos0 .. pos0 + s - 1 of the paged home `table`."""
    _cuda(table, k, v)
    if k.dim() == 4:
        k, v = k[0], v[0]
    Hk, s, D = k.shape
    rc = lib().lb2_kvh_put(_ptr(table), _ptr(k), i64(*k.stride()), _ptr(v), i64(*v.stride()), int(pos0), s, Hk, D,
                           dtype_code(k), int(logc), _stream(k))
    check(rc, "kvh_put")


def kvh_gather(table, tb, cr, n, Hk, D, dtype, logc, device):
    """The QSA picks of a sequence of n positions read from the paged home: kg, vg [1, Hk, m, D]."""
    tb = tb.reshape(-1)
    nsel = tb.numel()
    m = nsel * cr + n - n // cr * cr
    kg = torch.empty((1, Hk, m, D), dtype=dtype, device=device)
    vg = torch.empty_like(kg)
    rc = lib().lb2_kvh_gather(_ptr(table), _ptr(tb), nsel, int(cr), int(n), _ptr(kg), _ptr(vg), Hk, D,
                              dtype_code(kg), int(logc), _stream(kg))
    check(rc, "kvh_gather")
    return kg, vg


def kvh_lru_plan(tb, lru):
    """One token's plan over the LRU state `lru` (a kv_host.Lru): sl [nsel] int32 on the device, the state updated in
    place (see lb2_kvh_lru_plan)."""
    tb = tb.reshape(-1)
    _cuda(tb, lru.slot_of)
    if tb.dtype != torch.int32:
        raise ValueError("kvh_lru_plan: tb must be int32")
    sl = torch.empty(tb.numel(), dtype=torch.int32, device=tb.device)
    rc = lib().lb2_kvh_lru_plan(_ptr(tb), tb.numel(), _ptr(lru.slot_of), lru.slot_of.numel(), _ptr(lru.block_of),
                                _ptr(lru.stamp), _ptr(lru.ref), _ptr(lru.meta), lru.slots, _ptr(sl), _stream(tb))
    check(rc, "kvh_lru_plan")
    return sl


def kvh_lru_gather(table, lru, tb, sl, cr, n, kn, vn, logc):
    """The token's QSA rows kg, vg [1, Hk, m, D] of a sequence of n positions through the LRU (pool hits, home
    misses filling their victims), and the new row kn / vn ([Hk, D], [1, Hk, 1, D] ...) written into the home at
    n - 1 (see lb2_kvh_lru_gather)."""
    tb = tb.reshape(-1)
    Hk, D = lru.pool.shape[2], lru.pool.shape[4]
    kn, vn = kn.reshape(Hk, D), vn.reshape(Hk, D)
    _cuda(table, tb, sl, kn, vn)
    if kn.dtype != lru.pool.dtype or vn.dtype != lru.pool.dtype:
        raise ValueError("kvh_lru_gather: the new row must have the pool's dtype")
    nsel = tb.numel()
    m = nsel * cr + n - n // cr * cr
    kg = torch.empty((1, Hk, m, D), dtype=kn.dtype, device=kn.device)
    vg = torch.empty_like(kg)
    rc = lib().lb2_kvh_lru_gather(_ptr(table), _ptr(lru.pool), lru.slots, _ptr(tb), _ptr(sl), nsel, int(cr), int(n),
                                  _ptr(kn), i64(*kn.stride()), _ptr(vn), i64(*vn.stride()), _ptr(kg), _ptr(vg), Hk, D,
                                  dtype_code(kg), int(logc), _stream(kg))
    check(rc, "kvh_lru_gather")
    return kg, vg


def kvh_lru_inval(lru, lim):
    """Slots of the LRU holding a block >= lim drop it."""
    rc = lib().lb2_kvh_lru_inval(_ptr(lru.slot_of), _ptr(lru.block_of), _ptr(lru.ref), lru.slots, int(lim),
                                 _stream(lru.slot_of))
    check(rc, "kvh_lru_inval")


# ---------------------------------------------------------------------------------------------------- GDN glue

def _rounded(x, dtype):
    """A Python float rounded to `dtype` (the scalar an op on that dtype applies)."""
    return float(torch.tensor(float(x), dtype=dtype).item())


def gdn_step_glue(conv, a, b, A_log, dt_bias, state, Hk, Dk, Hv, Dv):
    """Fused GDN decode rows (silu, q/k RMSNorm and scales, sigmoid(b), compute_g, recurrence) for B = 1."""
    _cuda(conv, a, b, A_log, dt_bias, state)
    NR = conv.shape[-2]
    conv, a, b = conv.reshape(NR, -1).contiguous(), a.reshape(NR, Hv).contiguous(), b.reshape(NR, Hv).contiguous()
    A_log, dt_bias = A_log.float().contiguous(), dt_bias.float().contiguous()
    state = state.contiguous()
    y = torch.empty((1, NR, Hv, Dv), dtype=conv.dtype, device=conv.device)
    s_out = torch.empty_like(state)
    inv = Dk ** -0.5
    rc = lib().lb2_gdn_step_glue(_ptr(conv), _ptr(a), _ptr(b), _ptr(A_log), _ptr(dt_bias), _ptr(state), _ptr(s_out),
                                 _ptr(y), NR, Hk, Dk, Hv, Dv, dtype_code(conv), _rounded(inv * inv, conv.dtype),
                                 _rounded(inv, conv.dtype), float(1e-6 * inv * inv), _stream(conv))
    check(rc, "gdn_step_glue")
    return y, s_out


def gdn_norm_gate(x, z, weight, eps):
    """silu(z) * (weight * rms_norm(x)) over the last axis."""
    _cuda(x, z, weight)
    D = x.shape[-1]
    xc, zc = x.contiguous(), z.contiguous()
    out = torch.empty_like(xc)
    rc = lib().lb2_gdn_norm_gate(_ptr(xc), _ptr(zc), _ptr(weight.contiguous()), _ptr(out), xc.numel() // D, D,
                                 dtype_code(xc), float(eps), _stream(xc))
    check(rc, "gdn_norm_gate")
    return out


# ---------------------------------------------------------------------------------------------------- paged 8-bit cache

# These calls are a few microseconds on the device, as much as Python needs for a dozen attribute reads: each reads what it
# checks once and looks for the reason of a refusal only when there is one.

_LAYOUTS = {"half": 0, "interleaved": 1}
_E4M3, _I32, _I64, _FP32 = torch.float8_e4m3fn, torch.int32, torch.int64, torch.float32


def _interleaved(layout, what):
    try:
        return _LAYOUTS[layout]
    except (KeyError, TypeError):
        raise ValueError(f"{what}: layout must be 'half' or 'interleaved', got {layout!r}") from None


def _int32(t, shape, dev, what):
    if t.dtype is not _I32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous int32 {list(shape)} on the same device")


def _turns(turns, D, dev, what):
    R = 2 * turns.numel()
    if turns.dtype is not _I64 or turns.dim() != 1 or turns.get_device() != dev or not turns.is_contiguous():
        raise ValueError(f"{what}: turns must be contiguous int64 [R / 2] on the same device")
    if not 2 <= R <= D:
        raise ValueError(f"{what}: turns for 2 to {D} rotated dims (one a pair), got {R}")
    return R


def _new_like(x):
    """An uninitialised tensor like x [B, H, T, D] with a unit last stride, and its strides. (empty_like follows the order of
    x's strides, which for rows that overlap in memory may put D elsewhere.)"""
    out = torch.empty_like(x)
    st = out.stride()
    if st[3] != 1:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        st = out.stride()
    return out, st


def _out_like(out, x, what):
    if out.shape != x.shape or out.dtype is not x.dtype or out.get_device() != x.get_device() or out.stride(-1) != 1:
        raise ValueError(f"{what}: out must have the result's shape, dtype and device, and a unit last stride")


def rope(x, positions, turns, layout="half", amp=1.0, inverse=False, out=None):
    """x [B, H, T, D] with the first 2 * len(turns) dims of each head rotated by the rows' positions (lb2_rope).

    positions int32 [B, T] or [T]; turns int64 [R / 2] (larder_b200.rope.Rope(...).turns); layout "half" (pairs i,
    i + R / 2) or "interleaved" (2 i, 2 i + 1); inverse=True is the gradient, which autograd takes where x asks for one.
    out may be x."""
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("rope: out= does not take part in a graph; x requires a gradient")
        return _Rope.apply(x, positions, turns, layout, amp, inverse)
    dev, st = x.get_device(), x.stride()
    if dev < 0:
        _cuda(x)
    if len(st) != 4 or st[3] != 1:
        raise ValueError("rope: x must be [B, H, T, D] with a unit last stride")
    B, H, T, D = x.shape
    R = _turns(turns, D, dev, "rope")
    ps = positions.shape
    _int32(positions, (T,) if len(ps) == 1 else (B, T), dev, "rope: positions")
    if out is None:
        out, ost = _new_like(x)
    else:
        _out_like(out, x, "rope")
        ost = out.stride()
        if out.data_ptr() == x.data_ptr() and ost != st:
            raise ValueError("rope: out over x must have x's strides")
    rc = lib().lb2_rope(x.data_ptr(), i64(*st[:3]), out.data_ptr(), i64(*ost[:3]), positions.data_ptr(),
                        0 if len(ps) == 1 else T, turns.data_ptr(), B, H, T, D, R, dtype_code(x),
                        _interleaved(layout, "rope"), 1 if inverse else 0, amp, _stream_of(dev))
    if rc:
        check(rc, "rope")
    return out


class _Rope(torch.autograd.Function):
    """rope in autograd's graph: the gradient is the transposed map, the inverse rotation with the same amp."""

    @staticmethod
    def forward(ctx, x, positions, turns, layout, amp, inverse):
        ctx.save_for_backward(positions, turns)
        ctx.how = layout, amp, inverse
        return rope(x, positions, turns, layout, amp, inverse)

    @staticmethod
    def backward(ctx, dy):
        layout, amp, inverse = ctx.how
        if dy.stride(-1) != 1:
            dy = dy.contiguous()
        return rope(dy, *ctx.saved_tensors, layout, amp, not inverse), None, None, None, None, None


def _kv8_pool(pages, scales, table, what):
    """(pages' shape, table's shape, device index) of a checked pool."""
    ps, ts, dev = pages.shape, table.shape, pages.get_device()
    if dev < 0:
        _cuda(pages)
    if len(ps) != 5 or ps[1] != 2 or pages.dtype is not _E4M3 or not pages.is_contiguous():
        raise ValueError(f"{what}: pages must be contiguous float8_e4m3fn [num_pages, 2, Hkv, page, D]")
    if scales.dtype is not _FP32 or scales.shape != ps[:3] or scales.get_device() != dev or not scales.is_contiguous():
        raise ValueError(f"{what}: scales must be contiguous fp32 [num_pages, 2, Hkv] on the pages' device")
    if table.dtype is not _I32 or len(ts) != 2 or table.get_device() != dev or table.stride(1) != 1:
        raise ValueError(f"{what}: table must be int32 [B, max_pages] with a unit last stride on the pages' device")
    return ps, ts, dev


_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _elsewhere(dev, call, *args):
    """A call for tensors of another device than the current one, made there."""
    with torch.cuda.device(dev):
        return call(*args)


def kv8_append(pages, scales, k, v, table, start, lens=None, cu=None, turns=None, layout="half", amp=1.0):
    """Appends k / v [B, Hkv, T, D] to the paged 8-bit cache in place (lb2_kv8_append): sequence b's tokens become its
    positions start[b] onwards (start int32 [B]), keys rotated by them when turns is given. lens int32 [B]: only the
    first lens[b] tokens of each. cu int32 [B + 1]: k / v are [1, Hkv, T, D] and sequence b's tokens are rows cu[b] to
    cu[b + 1] - 1."""
    (num_pages, _, Hkv, page, D), (B, max_pages), dev = _kv8_pool(pages, scales, table, "kv8_append")
    if dev != _device():
        return _elsewhere(dev, kv8_append, pages, scales, k, v, table, start, lens, cu, turns, layout, amp)
    ks, kst, vst = k.shape, k.stride(), v.stride()
    if (len(ks) != 4 or ks != v.shape or k.dtype is not v.dtype or k.get_device() != dev or v.get_device() != dev
            or kst[3] != 1 or vst[3] != 1):
        raise ValueError("kv8_append: k and v must share shape, dtype and the cache's device, with unit last strides")
    T = ks[2]
    if ks[0] != (B if cu is None else 1) or ks[1] != Hkv or ks[3] != D:
        raise ValueError("kv8_append: k / v must be [B, Hkv, T, D] for the table's B and the cache's Hkv and D "
                         "([1, Hkv, T, D] with cu)")
    _int32(start, (B,), dev, "kv8_append: start")
    if lens is not None:
        _int32(lens, (B,), dev, "kv8_append: lens")
    if cu is not None:
        _int32(cu, (B + 1,), dev, "kv8_append: cu")
    R = 0 if turns is None else _turns(turns, D, dev, "kv8_append")
    rc = lib().lb2_kv8_append(pages.data_ptr(), scales.data_ptr(), k.data_ptr(), i64(*kst[:3]), v.data_ptr(),
                              i64(*vst[:3]), table.data_ptr(), table.stride(0), start.data_ptr(), _ptr(lens), _ptr(cu),
                              _ptr(turns), B, Hkv, T, D, R, page, num_pages, max_pages, dtype_code(k),
                              _interleaved(layout, "kv8_append"), amp, _stream_of(dev))
    if rc:
        check(rc, "kv8_append")


_KV8_WS = {}  # (B, Hq, Hkv, T, D, page, max_pages, device index) -> workspace bytes


def kv8_attend(q, pages, scales, table, kv_len, scale, causal=True, out=None):
    """Attention of q [B, Hq, T, D] over each sequence's first kv_len[b] cached tokens (lb2_kv8_attend); kv_len int32
    [B] counts the call's own tokens, which are already appended. causal: row t sees keys 0 .. kv_len - T + t. For
    inference: the result is in no autograd graph."""
    (num_pages, _, Hkv, page, D), (B, max_pages), dev = _kv8_pool(pages, scales, table, "kv8_attend")
    if dev != _device():
        return _elsewhere(dev, kv8_attend, q, pages, scales, table, kv_len, scale, causal, out)
    qs, qst = q.shape, q.stride()
    if len(qs) != 4 or qs[0] != B or qs[3] != D or q.get_device() != dev or qst[3] != 1:
        raise ValueError("kv8_attend: q must be [B, Hq, T, D] for the table's B and the cache's D and device, with a unit "
                         "last stride")
    Hq, T = qs[1], qs[2]
    if Hq == 0 or Hq % Hkv:
        raise ValueError("kv8_attend: Hq must be a multiple of the cache's Hkv")
    _int32(kv_len, (B,), dev, "kv8_attend: kv_len")
    if out is None:
        out, ost = _new_like(q)
    else:
        _out_like(out, q, "kv8_attend")
        ost = out.stride()
    key = (B, Hq, Hkv, T, D, page, max_pages, dev)
    n = _KV8_WS.get(key)
    if n is None:
        n = _KV8_WS[key] = lib().lb2_kv8_attend_workspace_size(*key[:7])
    stream = _stream_of(dev)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_kv8_attend(q.data_ptr(), i64(*qst[:3]), pages.data_ptr(), scales.data_ptr(), table.data_ptr(),
                                  table.stride(0), kv_len.data_ptr(), out.data_ptr(), i64(*ost[:3]), B, Hq, Hkv,
                                  T, D, page, num_pages, max_pages, dtype_code(q), scale, 1 if causal else 0, ws, n, stream)
    finally:
        _scratch_done(ws)
    if rc:
        check(rc, "kv8_attend")
    return out


def kv8_attend_packed(q, pages, scales, table, kv_len, cu, scale, causal=True, out=None):
    """Attention of packed chunks of new tokens over the paged 8-bit cache (lb2_kv8_attend_packed): q [1, Hq, T, D], sequence
    b's rows cu[b] .. cu[b + 1] - 1 (cu int32 [B + 1]) being the last of its kv_len[b] cached tokens (int32 [B], the call's
    own among them, already appended). causal: each row sees the tokens up to its own. For inference: the result is in no
    autograd graph. out must not overlap q."""
    (num_pages, _, Hkv, page, D), (B, max_pages), dev = _kv8_pool(pages, scales, table, "kv8_attend_packed")
    if dev != _device():
        return _elsewhere(dev, kv8_attend_packed, q, pages, scales, table, kv_len, cu, scale, causal, out)
    qs, qst = q.shape, q.stride()
    if len(qs) != 4 or qs[0] != 1 or qs[3] != D or q.get_device() != dev or qst[3] != 1:
        raise ValueError("kv8_attend_packed: q must be [1, Hq, T, D] for the cache's D and device, with a unit last stride")
    Hq, T = qs[1], qs[2]
    if Hq == 0 or Hq % Hkv:
        raise ValueError("kv8_attend_packed: Hq must be a multiple of the cache's Hkv")
    _int32(kv_len, (B,), dev, "kv8_attend_packed: kv_len")
    _int32(cu, (B + 1,), dev, "kv8_attend_packed: cu")
    if out is None:
        out, ost = _new_like(q)
    else:
        _out_like(out, q, "kv8_attend_packed")
        ost = out.stride()
        if T and out.data_ptr() == q.data_ptr():
            raise ValueError("kv8_attend_packed: out must not be q's memory (some rows are read a second time)")
    n = lib().lb2_kv8_attend_packed_workspace_size(B, Hq, Hkv, T, D)
    stream = _stream_of(dev)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_kv8_attend_packed(q.data_ptr(), i64(*qst[1:3]), pages.data_ptr(), scales.data_ptr(),
                                         table.data_ptr(), table.stride(0), kv_len.data_ptr(), cu.data_ptr(),
                                         out.data_ptr(), i64(*ost[1:3]), B, Hq, Hkv, T, D, page, num_pages, max_pages,
                                         dtype_code(q), scale, 1 if causal else 0, ws, n, stream)
    finally:
        _scratch_done(ws)
    if rc:
        check(rc, "kv8_attend_packed")
    return out


def kv8_copy(pages, scales, src, dst, into=None):
    """Copies pages, codes and scales, in place: page dst[i] becomes page src[i] (int32 [n] on the device; lb2_kv8_copy).
    into: (pages, scales) of another pool of the same heads, page and D, whose pages dst names. No page may be in dst
    twice, nor, within one pool, in both src and dst."""
    ps, dev = pages.shape, pages.get_device()
    to, to_scales = (pages, scales) if into is None else into
    for p, s in ((pages, scales), (to, to_scales)) if into is not None else ((pages, scales),):
        if p.get_device() < 0:
            _cuda(p)
        if len(p.shape) != 5 or p.shape[1:] != ps[1:] or ps[1] != 2 or p.dtype is not _E4M3 or not p.is_contiguous():
            raise ValueError("kv8_copy: pools must be contiguous float8_e4m3fn [num_pages, 2, Hkv, page, D], of one Hkv, page "
                             "and D")
        if s.dtype is not _FP32 or s.shape != p.shape[:3] or not s.is_contiguous():
            raise ValueError("kv8_copy: scales must be contiguous fp32 [num_pages, 2, Hkv]")
        if p.get_device() != dev or s.get_device() != dev:
            raise ValueError("kv8_copy: the pools must be on one device")
    if dev != _device():
        return _elsewhere(dev, kv8_copy, pages, scales, src, dst, into)
    n = src.numel()
    _int32(src, (n,), dev, "kv8_copy: src")
    _int32(dst, (n,), dev, "kv8_copy: dst")
    rc = lib().lb2_kv8_copy(pages.data_ptr(), scales.data_ptr(), ps[0], to.data_ptr(), to_scales.data_ptr(), to.shape[0],
                            src.data_ptr(), dst.data_ptr(), n, ps[2], ps[3], ps[4], _stream_of(dev))
    if rc:
        check(rc, "kv8_copy")


def kv8_compact(pages, scales, table, keep, cu, to, start, turns=None, layout="half"):
    """Moves kept tokens of paged sequences together, in place (lb2_kv8_compact): the tokens at positions keep[cu[b]] ..
    keep[cu[b + 1] - 1] of sequence b (keep int32 [T], cu int32 [B + 1]) become its positions start[b] onwards (start int32
    [B], page beginnings) in the pages to[b] (int32 [B, max_to], entry j for positions j * page and on), keys turned by the
    difference of the positions when turns is given. No page may be written twice, or both read and written."""
    (num_pages, _, Hkv, page, D), (B, max_pages), dev = _kv8_pool(pages, scales, table, "kv8_compact")
    if dev != _device():
        return _elsewhere(dev, kv8_compact, pages, scales, table, keep, cu, to, start, turns, layout)
    T, ts = keep.numel(), to.shape
    _int32(keep, (T,), dev, "kv8_compact: keep")
    _int32(cu, (B + 1,), dev, "kv8_compact: cu")
    _int32(start, (B,), dev, "kv8_compact: start")
    if to.dtype is not _I32 or len(ts) != 2 or ts[0] != B or to.get_device() != dev or to.stride(1) != 1:
        raise ValueError("kv8_compact: to must be int32 [B, max_to] with a unit last stride on the pages' device")
    R = 0 if turns is None else _turns(turns, D, dev, "kv8_compact")
    rc = lib().lb2_kv8_compact(pages.data_ptr(), scales.data_ptr(), table.data_ptr(), table.stride(0), keep.data_ptr(),
                               cu.data_ptr(), to.data_ptr(), to.stride(0), start.data_ptr(), _ptr(turns), B, Hkv, T, D, R,
                               page, num_pages, max_pages, ts[1], _interleaved(layout, "kv8_compact"), _stream_of(dev))
    if rc:
        check(rc, "kv8_compact")


def attn_packed(q, k, v, scale, cu, out=None):
    """Causal attention over prompts packed on one row axis (lb2_attn_packed): q [1, Hq, T, D], k / v [1, Hkv, T, D],
    cu int32 [S + 1] on the device, prompt s being rows cu[s] .. cu[s + 1] - 1. For inference: the result is in no autograd
    graph."""
    dev, qs, ks = q.get_device(), q.shape, k.shape
    qst, kst, vst = q.stride(), k.stride(), v.stride()
    if dev < 0:
        _cuda(q)
    if len(qs) != 4 or len(ks) != 4 or qs[0] != 1 or ks[0] != 1 or ks != v.shape:
        raise ValueError("attn_packed: q must be [1, Hq, T, D], k and v [1, Hkv, T, D]")
    if qst[3] != 1 or kst[3] != 1 or vst[3] != 1:
        raise ValueError("attn_packed: the last axis must have unit stride")
    _, Hq, T, D = qs
    Hkv = ks[1]
    if ks[2] != T or ks[3] != D or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError("attn_packed: q, k and v must share rows, head dim and dtype")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("attn_packed: q, k and v must share a device")
    S = cu.numel() - 1
    if S < 1:
        raise ValueError("attn_packed: cu must be int32 [S + 1], S >= 1")
    _int32(cu, (S + 1,), dev, "attn_packed: cu")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError("attn_packed: Hq must be a multiple of Hkv")
    if out is None:
        out, ost = _new_like(q)
    else:
        _out_like(out, q, "attn_packed")
        ost = out.stride()
    n = lib().lb2_attn_packed_workspace_size(S, Hq, Hkv, T, D)
    stream = _stream_of(dev)
    ws = _scratch(n or 1, stream)
    try:
        rc = lib().lb2_attn_packed(q.data_ptr(), i64(*qst[1:3]), k.data_ptr(), i64(*kst[1:3]), v.data_ptr(),
                                   i64(*vst[1:3]), out.data_ptr(), i64(*ost[1:3]), cu.data_ptr(), S, Hq, Hkv,
                                   T, D, dtype_code(q), scale, ws, n, stream)
    finally:
        _scratch_done(ws)
    if rc:
        check(rc, "attn_packed")
    return out
