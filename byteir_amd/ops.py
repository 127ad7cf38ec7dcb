"""Direct calls into the kernel C ABI with torch tensors as device memory.

torch is used for allocation and streams only; every computation below is a hand-written
HIP kernel reached through libbrt_rocm_kernels.so / libflash_attn.so.  Shapes follow the
reference's op kernels: reductions take the canonical [A, B, C] view computed by
`canonicalize_reduce` (ReduceImpl, runtime/lib/backends/cuda/providers/default/reduction/reduce_impl.h:28-59).
"""
import collections
import ctypes
import functools
import operator
import struct

import torch

from . import _lib

_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _dev(t):
    if not t.is_cuda:
        raise ValueError("device tensor required: the ROCm provider has no host path")
    if not t.is_contiguous():
        raise ValueError("dense row-major tensor required")
    return ctypes.c_void_p(t.data_ptr())


def fill(t, dist, seed, a=0.0, b=1.0, stream=None):
    """Counter-based synthetic data in place (brt_rocm_fill): element i is a function of
    (seed, i) only; dist = _lib.FILL_UNIFORM ([a, b)) or _lib.FILL_NORMAL (mean 0, sigma b)."""
    _lib.check(_lib.kernels().brt_rocm_fill(_DT[t.dtype], dist, seed, _dev(t), t.numel(), a, b, _stream(stream)),
               "brt_rocm_fill")
    return t


def deduce_output_shape(shape, dims):
    """reduction::DeduceOutputShape, runtime/lib/core/common/utils/math_helper.cc:145-159."""
    for d in dims:
        if not 0 <= d < len(shape):
            raise ValueError("invalid dimension")
    return [s for i, s in enumerate(shape) if i not in dims]


def canonicalize_reduce(in_shape, out_shape, dims):
    """ReduceImpl's constructor: -> (A, B, C); raises ValueError where the reference throws."""
    if list(out_shape) != deduce_output_shape(in_shape, dims):
        raise ValueError("output shape does not match the deduced shape")
    live = sorted(d for d in dims if in_shape[d] != 1)
    if not live:
        n = 1
        for s in in_shape:
            n *= s
        return 0, 0, n
    if any(b - a != 1 for a, b in zip(live, live[1:])):
        raise ValueError("Only consecutive dimensions reduction is supported")
    A = B = C = 1
    for s in in_shape[:live[0]]:
        A *= s
    for d in live:
        B *= in_shape[d]
    for s in in_shape[live[-1] + 1:]:
        C *= s
    return A, B, C


def reduce_workspace_bytes(dtype, A, B, C):
    return _lib.kernels().brt_rocm_reduce_workspace_bytes(_DT[dtype], A, B, C)


def reduce_abc(op, x, out, A, B, C, workspace=None, stream=None):
    """Enqueue out[a,c] = fold_b x[a,b,c]; `workspace` is a uint8 device tensor of at least
    reduce_workspace_bytes(...) bytes (allocated here when omitted)."""
    K = _lib.kernels()
    need = K.brt_rocm_reduce_workspace_bytes(_DT[x.dtype], A, B, C)
    if need and workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    ws_ptr = ctypes.c_void_p(workspace.data_ptr()) if workspace is not None else None
    ws_len = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _lib.check(K.brt_rocm_reduce(op, _DT[x.dtype], _dev(x), _dev(out), A, B, C, ws_ptr, ws_len,
                                 _stream(stream)), "brt_rocm_reduce")
    return out


def reduce_abc_static(op, x, out, A, B, C, stream=None):
    """The same fold through brt_rocm_reduce_static: split partials in the library's own device
    array, no allocation of any kind; raises when the fold needs more than that array holds."""
    _lib.check(_lib.kernels().brt_rocm_reduce_static(op, _DT[x.dtype], _dev(x), _dev(out), A, B, C,
                                                     _stream(stream)), "brt_rocm_reduce_static")
    return out


def reduce(op, x, dims, stream=None):
    """Reduce<Op>Op over `dims` of a dense tensor (op: _lib.REDUCE_SUM / MAX / MIN / PROD / MEAN /
    SUMSQR)."""
    out_shape = deduce_output_shape(list(x.shape), list(dims))
    A, B, C = canonicalize_reduce(list(x.shape), out_shape, list(dims))
    out = torch.empty(out_shape, dtype=x.dtype, device=x.device)
    return reduce_abc(op, x, out, A, B, C, stream=stream)


def softmax_workspace_bytes(x, axis=-1):
    """brt_rocm_softmax_workspace_bytes for softmax(x, axis=axis)."""
    axis = axis % x.dim()
    a, b, c = 1, x.shape[axis], 1
    for n in x.shape[:axis]:
        a *= n
    for n in x.shape[axis + 1:]:
        c *= n
    return _lib.kernels().brt_rocm_softmax_workspace_bytes(_DT[x.dtype], a, b, c)


def softmax(x, out=None, stream=None, axis=-1, workspace=None):
    """byteir.softmax over `axis` of a dense tensor (the last one by default).  workspace: the
    caller's scratch (uint8 device tensor of softmax_workspace_bytes) for the inner-axis split."""
    if out is None:
        out = torch.empty_like(x)
    axis = axis % x.dim()
    a, b, c = 1, x.shape[axis], 1
    for n in x.shape[:axis]:
        a *= n
    for n in x.shape[axis + 1:]:
        c *= n
    if workspace is not None:
        _lib.check(_lib.kernels().brt_rocm_softmax_axis_ws(_DT[x.dtype], _dev(x), _dev(out), a, b, c, _dev(workspace),
                                                           workspace.numel() * workspace.element_size(), _stream(stream)),
                   "brt_rocm_softmax_axis_ws")
        return out
    _lib.check(_lib.kernels().brt_rocm_softmax_axis(_DT[x.dtype], _dev(x), _dev(out), a, b, c,
                                                    _stream(stream)), "brt_rocm_softmax_axis")
    return out


# ---- flash attention through the custom-library ABI ---------------------------------------
def round_up(x, m):
    return (x + m - 1) // m * m


def pack_flash_args(q, k, v, o, scale, window, p_dropout=0.0):
    """The 192-byte extra_args blob for [b, s, h, d] tensors: 17 i64, f32, 4 i64, f32, 2 i64,
    unpadded (OpAccessor::GetAttrAsVoidPtr, runtime/lib/core/framework/op_accessor.cc:212-242;
    field order compiler/lib/Conversion/HloToByreTensor/HloToByreCustom.cpp:149-176)."""
    b, sq, h, d = q.shape
    sk, h_k = k.shape[1], k.shape[2]
    ints1 = [q.stride(0), k.stride(0), v.stride(0), o.stride(0),
             q.stride(1), k.stride(1), v.stride(1), o.stride(1),
             q.stride(2), k.stride(2), v.stride(2), o.stride(2),
             b, h, h_k, d, round_up(d, 32)]
    ints2 = [sq, sk, round_up(sq, 128), round_up(sk, 128)]
    return (struct.pack("<17q", *ints1) + struct.pack("<f", scale) + struct.pack("<4q", *ints2)
            + struct.pack("<f", p_dropout) + struct.pack("<2q", *window))


def _call_custom(fn, tensors, blob, stream):
    arr = (ctypes.c_void_p * len(tensors))(*[t.data_ptr() if t is not None else None for t in tensors])
    buf = ctypes.create_string_buffer(blob, len(blob))
    fn(arr, ctypes.cast(buf, ctypes.c_void_p), _stream(stream))


def _call_custom_ws(kind, dtype, tensors, blob, workspace, stream):
    """flash_attn_<kind>_ws: the error-returning entry point with the caller's scratch
    (`workspace`: a uint8 device tensor, or None)."""
    L = _lib.flash_attn()
    arr = (ctypes.c_void_p * len(tensors))(*[t.data_ptr() if t is not None else None for t in tensors])
    buf = ctypes.create_string_buffer(blob, len(blob))
    ws = ctypes.c_void_p(workspace.data_ptr()) if workspace is not None else None
    n = workspace.numel() * workspace.element_size() if workspace is not None else 0
    rc = getattr(L, f"flash_attn_{kind}_ws")(arr, ctypes.cast(buf, ctypes.c_void_p), 1 if dtype == torch.float16 else 2, ws, n, _stream(stream))
    if rc < 0:
        raise ValueError(L.flash_attn_last_error().decode())
    _lib.check(rc, f"flash_attn_{kind}_ws")


def flash_attn_workspace_bytes(kind, dtype, blob, dq_accum_bytes=0):
    """flash_attn_{fwd,bwd,kvcache}_workspace_bytes for an extra_args blob."""
    L = _lib.flash_attn()
    buf = ctypes.create_string_buffer(blob, len(blob))
    code = 1 if dtype == torch.float16 else 2
    if kind in ("bwd", "sink_bwd"):
        return getattr(L, f"flash_attn_{kind}_workspace_bytes")(ctypes.cast(buf, ctypes.c_void_p), code, dq_accum_bytes)
    return getattr(L, f"flash_attn_{kind}_workspace_bytes")(ctypes.cast(buf, ctypes.c_void_p), code)


def rng_state_tensor(seed, offset, device):
    """The rng_state operand of the attention calls: {seed, offset} as two 64-bit words."""
    to_i64 = lambda x: int(x) - (1 << 64) if int(x) >= (1 << 63) else int(x)
    return torch.tensor([to_i64(seed), to_i64(offset)], dtype=torch.int64, device=device)


def flash_attn_fwd(q, k, v, scale, window=(-1, -1), stream=None, out=None, p_dropout=0.0, rng_state=None, workspace=None):
    """run_flash_attn_fwd: tensors {q, k, v, rng_state, o, softmax_lse, softmax_P}
    (external_libs/runtime/flash_attn/lib/flash_api.cu:586-654). -> (o, lse[b,h,sq] f32).
    out: optional (o, lse, rng_state) to write into instead of allocating.
    p_dropout > 0 reads {seed, offset} from rng_state (an int64[2] device tensor, see
    rng_state_tensor), as the reference's kernel does (flash_fwd_kernel.h:46-47)."""
    L = _lib.flash_attn()
    b, sq, h, d = q.shape
    if out is not None:
        o, lse, rng = out
    else:
        o = torch.empty_like(q)
        lse = torch.empty((b, h, sq), dtype=torch.float32, device=q.device)
        rng = rng_state if rng_state is not None else torch.zeros(2, dtype=torch.int64, device=q.device)
    blob = pack_flash_args(q, k, v, o, scale, window, p_dropout)
    if workspace is not None:  # the caller's scratch for the key-axis split (flash_attn_fwd_ws)
        _call_custom_ws("fwd", q.dtype, [q, k, v, rng, o, lse, None], blob, workspace, stream)
        return o, lse
    fn = L.run_flash_attn_fwd if q.dtype == torch.float16 else L.run_flash_attn_fwd_bf16
    _call_custom(fn, [q, k, v, rng, o, lse, None], blob, stream)
    return o, lse


def flash_attn_bwd_buffers(q, k, v):
    """The output and scratch tensors of run_flash_attn_bwd for these shapes:
    (dq, dk, dv, d_softmax, dq_accum, rng_state)."""
    b, sq, h, d = q.shape
    sq_r, d_r = round_up(sq, 128), round_up(d, 32)
    like = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device)
    # dq, dk, dv are addressed with the strides of q, k, v (flash_api.cu:377-389)
    return (like(q), like(k), like(v),
            torch.empty((b, h, sq_r), dtype=torch.float32, device=q.device),
            torch.empty((b, sq_r, h, d_r), dtype=torch.float32, device=q.device),
            torch.zeros(2, dtype=torch.int64, device=q.device))


def flash_attn_bwd(dout, q, k, v, o, lse, scale, window=(-1, -1), stream=None, out=None, p_dropout=0.0,
                   rng_state=None, workspace=None):
    """run_flash_attn_bwd: tensors {dout, q, k, v, out, softmax_lse, rng_state, dq, dk, dv,
    d_softmax, dq_accum} (flash_api.cu:656-725). -> (dq, dk, dv).
    out: optional result of flash_attn_bwd_buffers to write into instead of allocating.
    p_dropout > 0 needs the rng_state the forward call used."""
    L = _lib.flash_attn()
    dq, dk, dv, dsm, dq_accum, rng = out if out is not None else flash_attn_bwd_buffers(q, k, v)
    if rng_state is not None:
        rng = rng_state
    blob = pack_flash_args(q, k, v, o, scale, window, p_dropout)
    if workspace is not None:  # the caller's scratch for partial dK / dV (flash_attn_bwd_ws)
        _call_custom_ws("bwd", q.dtype, [dout, q, k, v, o, lse, rng, dq, dk, dv, dsm, dq_accum], blob, workspace, stream)
        return dq, dk, dv
    fn = L.run_flash_attn_bwd if q.dtype == torch.float16 else L.run_flash_attn_bwd_bf16
    _call_custom(fn, [dout, q, k, v, o, lse, rng, dq, dk, dv, dsm, dq_accum], blob, stream)
    return dq, dk, dv


def pack_flash_kvcache_args(q, kcache, vcache, knew, vnew, o, scale, window):
    """The 244-byte extra_args blob of run_flash_attn_kvcache: 24 i64, f32, 6 i64, unpadded
    (field order external_libs/runtime/flash_attn/lib/flash_api.cu:727-773).  knew / vnew may
    be None: their strides and seqlen_knew are then 0."""
    b, sq, h, d = q.shape
    sk, h_k = kcache.shape[1], kcache.shape[2]
    kn = knew if knew is not None else None
    st = lambda t, i: t.stride(i) if t is not None else 0
    ints1 = [q.stride(0), kcache.stride(0), vcache.stride(0), st(kn, 0), st(vnew, 0), o.stride(0),
             q.stride(1), kcache.stride(1), vcache.stride(1), st(kn, 1), st(vnew, 1), o.stride(1),
             q.stride(2), kcache.stride(2), vcache.stride(2), st(kn, 2), st(vnew, 2), o.stride(2),
             b, h, h_k, d, round_up(d, 32), knew.shape[1] if knew is not None else 0]
    ints2 = [sq, sk, round_up(sq, 128), round_up(sk, 128), window[0], window[1]]
    return struct.pack("<24q", *ints1) + struct.pack("<f", scale) + struct.pack("<6q", *ints2)


def flash_attn_kvcache(q, kcache, vcache, knew, vnew, seqlens_k, scale, window=(-1, -1), stream=None, workspace=None):
    """run_flash_attn_kvcache: tensors {q, k_cache, v_cache, k_new, v_new, seqlens_k, o,
    softmax_lse} (flash_api.cu:727-811).  Appends knew / vnew to the caches IN PLACE at row
    seqlens_k[b], then attends to the first seqlens_k[b] + seqlen_knew rows of each batch.
    seqlens_k: int32 [b] device tensor. -> (o, lse[b,h,sq] f32)."""
    L = _lib.flash_attn()
    b, sq, h, d = q.shape
    o = torch.empty_like(q)
    lse = torch.empty((b, h, sq), dtype=torch.float32, device=q.device)
    blob = pack_flash_kvcache_args(q, kcache, vcache, knew, vnew, o, scale, window)
    if workspace is not None:
        _call_custom_ws("kvcache", q.dtype, [q, kcache, vcache, knew, vnew, seqlens_k, o, lse], blob, workspace, stream)
        return o, lse
    fn = L.run_flash_attn_kvcache if q.dtype == torch.float16 else L.run_flash_attn_kvcache_bf16
    _call_custom(fn, [q, kcache, vcache, knew, vnew, seqlens_k, o, lse], blob, stream)
    return o, lse


# ---- attention with a window and sinks, over a paged cache, and eviction from a cache -----------
# A call is checked, its blob packed and its scratch asked for once per set of shapes, strides, types
# and scalars (the _plan_* functions, memoised on exactly those: nothing of a tensor's contents or
# address); what is left per call is the outputs, the pointers and the launch.  One decode step or
# short prompt takes the GPU 10-15 us, checks and packing took the host 25-45 us.
_PLANS = 4096  # plans kept; serving sees one per batch shape, training one per sequence length
_Sig = collections.namedtuple("_Sig", "shape stride dtype device")


def _nums(scale, *ints):
    """The scalars of a call as Python numbers: a plan is memoised on their values, and a 0-d tensor in their
    place would be memoised by its identity."""
    return float(scale), *map(operator.index, ints)


def _window(window):
    left, right = window
    return operator.index(left), operator.index(right)


def _sig(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _fresh(shape, dtype, device):
    """The signature of a dense tensor that the call itself makes."""
    stride, n = [], 1
    for x in reversed(shape):
        stride.insert(0, n)
        n *= max(x, 1)
    return _Sig(torch.Size(shape), tuple(stride), dtype, device)


def _sigs(*sigs):
    return [None if s is None else _Sig(*s) for s in sigs]


def _on(device, *sigs):
    """Everything lies on one GPU."""
    if device < 0:
        raise ValueError("device tensor required: the ROCm provider has no host path")
    for t in sigs:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on devices {device} and {t.device}: one call takes tensors of one GPU")


def _like(t, dtype, shape, what):
    if t is not None and (t.dtype != dtype or tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{what} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _dense(t, what):
    n = 1
    for size, stride in zip(reversed(t.shape), reversed(t.stride)) if t is not None and 0 not in t.shape else ():
        if size != 1 and stride != n:
            raise ValueError(f"{what} must be dense row-major")
        n *= size


def _half(q, *sigs):
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{q.dtype} is not supported (float16 or bfloat16)")
    for t in sigs:
        if t is not None and t.dtype != q.dtype:
            raise ValueError(f"tensors of {q.dtype} and {t.dtype}: one call takes one storage type")
    for t in (q,) + sigs:
        if t is not None and (len(t.shape) != 4 or (0 not in t.shape and t.shape[3] > 1 and t.stride[3] != 1)):
            raise ValueError("4-d tensors with a dense head_dim required")


def _strides(t):
    """(outer, row, head) strides; an axis of length 1 has none that counts."""
    return [t.stride[i] if t.shape[i] > 1 else 0 for i in range(3)] if t is not None else [0, 0, 0]


def _overlaps(t):
    """Whether elements of a view may share memory (an expanded axis, say)."""
    end = 0
    for stride, n in sorted((s, n) for s, n in zip(t.stride, t.shape) if n > 1):
        if stride <= end:
            return True
        end += stride * (n - 1)
    return False


def _plan(kind, dtype, blob, dq_accum_bytes=0):
    """What a call needs besides pointers: (entry point, blob, storage type, scratch bytes)."""
    return _lib.flash_attn_entry(kind), blob, 1 if dtype == torch.float16 else 2, flash_attn_workspace_bytes(kind, dtype, blob, dq_accum_bytes)


_pack11 = struct.Struct("11P").pack
_pack12 = struct.Struct("12P").pack


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _on_stream(fn):
    """Runs a call with stream=... under that stream, so that what it allocates belongs to it."""
    @functools.wraps(fn)
    def call(*args, stream=None, **kw):
        if stream is None:
            return fn(*args, **kw)
        first = args[0] if args else kw[fn.__code__.co_varnames[0]]
        if stream.device != first.device:
            raise ValueError(f"a stream of {stream.device} for tensors of {first.device}")
        with torch.cuda.stream(stream):
            return fn(*args, **kw)
    return call


def _launch(plan, tensors, on, workspace):
    """The call on the GPU of `on` and its current stream, with the caller's scratch or scratch from torch's
    allocator; raises ValueError for a call that the library refuses."""
    entry, blob, code, need = plan
    device = on.get_device()
    if torch.cuda.current_device() != device:
        with torch.cuda.device(device):
            return _launch(plan, tensors, on, workspace)
    ws, n = 0, 0
    if workspace is not None:
        if workspace.get_device() != device:
            raise ValueError("the workspace must lie on the tensors' GPU")
        if not workspace.is_contiguous():  # its bytes are counted by its elements
            raise ValueError("the workspace must be dense")
        ws, n = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=on.device)
        ws, n = workspace.data_ptr(), need
    rc = entry(tensors, blob, code, ws, n, torch.cuda.current_stream().cuda_stream)
    if rc < 0:
        raise ValueError(_lib.flash_attn().flash_attn_last_error().decode())
    _lib.check(rc, "flash_attn")


def pack_flash_sink_args(q, k, v, o, scale, window, n_sink):
    """The 200-byte extra_args blob of flash_attn_sink_fwd / _bwd: pack_flash_args, then i64 n_sink."""
    return pack_flash_args(q, k, v, o, scale, window) + struct.pack("<q", n_sink)


def _sink_blob(q, k, v, o, scale, window, n_sink):
    """pack_flash_sink_args from signatures."""
    _half(q, k, v, o)
    b, sq, h, d = q.shape
    sk = k.shape[1]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    _like(o, q.dtype, q.shape, "o")
    each = [_strides(t) for t in (q, k, v, o)]
    return (struct.pack("<17q", *[s[i] for i in range(3) for s in each], b, h, k.shape[2], d, round_up(d, 32)) + struct.pack("<f", scale)
            + struct.pack("<4q", sq, sk, round_up(sq, 128), round_up(sk, 128)) + struct.pack("<f", 0.0) + struct.pack("<3q", *window, n_sink))


@functools.lru_cache(_PLANS)
def _plan_sink_fwd(q, k, v, o, lse, scale, window, n_sink):
    q, k, v, o, lse = _sigs(q, k, v, o, lse)
    _half(q)
    b, sq, h, _ = q.shape
    o = o or _fresh(q.shape, q.dtype, q.device)
    lse = lse or _fresh((b, h, sq), torch.float32, q.device)
    blob = _sink_blob(q, k, v, o, scale, window, n_sink)
    _like(lse, torch.float32, (b, h, sq), "lse")
    _dense(lse, "lse")
    if _overlaps(o):
        raise ValueError("o must not be a broadcast view")
    _on(q.device, k, v, o, lse)
    return _plan("sink_fwd", q.dtype, blob)


@_on_stream
def flash_attn_sink_fwd(q, k, v, scale, window=(-1, 0), n_sink=0, out=None, workspace=None):
    """Attention in which row i sees the keys of its window, as in flash_attn_fwd, and of the first
    `n_sink` keys those that the window's right side admits: q [b, sq, h, d], k, v [b, sk, h_k, d]
    -> (o [b, sq, h, d], lse [b, h, sq] f32).  lse comes from unrounded fp32 sums at every
    head_dim.  A row that sees no key gives o = 0, lse = +inf.  A key that no row of a 256-row
    block sees may hold anything; a NaN in a key that some row sees may reach the rows beside it.
    out: optional (o, lse) to write into; workspace: optional uint8 device tensor of
    flash_attn_workspace_bytes("sink_fwd", ...) bytes; stream: runs there, not on the current stream
    (these three are keywords of the calls below too)."""
    o, lse = out if out is not None else (None, None)
    scale, n_sink = _nums(scale, n_sink)
    plan = _plan_sink_fwd(_sig(q), _sig(k), _sig(v), _sig(o), _sig(lse), scale, _window(window), n_sink)
    if out is None:
        b, sq, h, _ = q.shape
        o, lse = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty((b, h, sq), dtype=torch.float32, device=q.device)
    _launch(plan, _pack11(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, o.data_ptr(), lse.data_ptr(), 0, 0, 0, 0, 0), q, workspace)
    return o, lse


@functools.lru_cache(_PLANS)
def _plan_sink_bwd(dout, q, k, v, o, lse, dq, dk, dv, dsm, dq_accum, scale, window, n_sink):
    """-> None when dout has to be laid out as o, or a broadcast input densely, before the call."""
    dout, q, k, v, o, lse, dq, dk, dv, dsm, dq_accum = _sigs(dout, q, k, v, o, lse, dq, dk, dv, dsm, dq_accum)
    blob = _sink_blob(q, k, v, o, scale, window, n_sink)
    _half(q, dout)
    b, sq, h, d = q.shape
    _like(dout, q.dtype, q.shape, "dout")
    _like(lse, torch.float32, (b, h, sq), "lse")
    _dense(lse, "lse")
    _on(q.device, dout, k, v, o, lse)
    if _strides(dout) != _strides(o) or any(_overlaps(t) for t in (q, k, v)):
        return None
    if dq is not None:
        for g, t, what in ((dq, q, "dq"), (dk, k, "dk"), (dv, v, "dv")):
            _like(g, t.dtype, t.shape, what)
            if _strides(g) != _strides(t):
                raise ValueError(f"{what} must be laid out as {what[1:]}")
        _like(dsm, torch.float32, (b, h, round_up(sq, 128)), "d_softmax")
        _dense(dsm, "d_softmax")
        _like(dq_accum, torch.float32, (b, round_up(sq, 128), h, round_up(d, 32)), "dq_accum")
        _dense(dq_accum, "dq_accum")
        _on(q.device, dq, dk, dv, dsm, dq_accum)
    accum = 4 * b * round_up(sq, 128) * h * round_up(d, 32) if dq_accum is not None else 0
    return _plan("sink_bwd", q.dtype, blob, accum)


@_on_stream
def flash_attn_sink_bwd(dout, q, k, v, o, lse, scale, window=(-1, 0), n_sink=0, out=None, workspace=None):
    """Gradients of flash_attn_sink_fwd -> (dq, dk, dv), laid out as q, k, v (densely where one is a
    broadcast view); dk and dv of a key/value head are the sums over its query heads.  o and lse
    are the forward call's.  out: optional (dq, dk, dv, d_softmax, dq_accum, _) of
    flash_attn_bwd_buffers; without it the partial sums of grouped heads go into the workspace."""
    dq, dk, dv, dsm, dq_accum, _ = out if out is not None else (None,) * 6
    scale, n_sink = _nums(scale, n_sink)
    key = (_sig(lse), _sig(dq), _sig(dk), _sig(dv), _sig(dsm), _sig(dq_accum), scale, _window(window), n_sink)
    plan = _plan_sink_bwd(_sig(dout), _sig(q), _sig(k), _sig(v), _sig(o), *key)
    if plan is None:
        # the library addresses dout with the strides of o, and the gradients with those of q, k, v
        o, q, k, v = (t.contiguous() if _overlaps(_Sig(*_sig(t))) else t for t in (o, q, k, v))
        if _strides(_Sig(*_sig(dout))) != _strides(_Sig(*_sig(o))):
            dout = torch.empty_strided(o.shape, o.stride(), dtype=o.dtype, device=o.device).copy_(dout)
        plan = _plan_sink_bwd(_sig(dout), _sig(q), _sig(k), _sig(v), _sig(o), *key)
    if out is None:
        dq, dk, dv = (torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device) for t in (q, k, v))
        dsm = torch.empty((q.shape[0], q.shape[2], round_up(q.shape[1], 128)), dtype=torch.float32, device=q.device)
    _launch(plan, _pack12(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), 0, dq.data_ptr(), dk.data_ptr(),
                          dv.data_ptr(), dsm.data_ptr(), _ptr(dq_accum)), q, workspace)
    return dq, dk, dv


def pack_flash_paged_args(q, k_pages, v_pages, k_new, v_new, o, scale, window, n_sink, max_pages, weights):
    """The 252-byte extra_args blob of flash_attn_paged: 18 strides in the order of the kvcache blob (the
    caches' outer stride is that of a page), i64 b, h, h_k, d, seqlen_knew; f32 scale; i64 seqlen_q,
    num_pages, page_size, max_pages, window left, right, n_sink, weights (0 none, 1 from zero, 2 on top
    of weights)."""
    return _paged_blob(*_sigs(*(_sig(t) for t in (q, k_pages, v_pages, k_new, v_new, o))), scale, window, n_sink, max_pages, weights)


def _paged_blob(q, k_pages, v_pages, k_new, v_new, o, scale, window, n_sink, max_pages, weights):
    b, sq, h, d = q.shape
    each = [_strides(t) for t in (q, k_pages, v_pages, k_new, v_new, o)]
    ints1 = [s[i] for i in range(3) for s in each] + [b, h, k_pages.shape[2], d, k_new.shape[1] if k_new is not None else 0]
    ints2 = [sq, k_pages.shape[0], k_pages.shape[1], max_pages, window[0], window[1], n_sink, weights]
    return struct.pack("<23q", *ints1) + struct.pack("<f", scale) + struct.pack("<8q", *ints2)


def _table(t, pages, b, what):
    """Checks a block table (or its absence) -> (max_pages, rows a sequence can hold)."""
    if t is None:
        if pages.shape[0] != b:
            raise ValueError(f"{b} sequences, but a dense cache of {pages.shape[0]}")
        return 0, pages.shape[1]
    if len(t.shape) != 2 or t.shape[1] == 0:
        raise ValueError(f"{what} must be [b, max_pages] with at least one page")
    _like(t, torch.int32, (b, t.shape[1]), what)
    _dense(t, what)
    return t.shape[1], t.shape[1] * pages.shape[1]


@functools.lru_cache(_PLANS)
def _plan_paged(q, k_pages, v_pages, block_table, seqlens_k, k_new, v_new, weights, weights_out, o, lse, scale, window, n_sink):
    q, k_pages, v_pages, block_table, seqlens_k, k_new, v_new, weights, weights_out, o, lse = _sigs(
        q, k_pages, v_pages, block_table, seqlens_k, k_new, v_new, weights, weights_out, o, lse)
    _half(q, k_pages, v_pages, k_new, v_new, o)
    b, sq, h, d = q.shape
    hk = k_pages.shape[2]
    if k_pages.shape != v_pages.shape or k_pages.shape[3] != d:
        raise ValueError(f"q {tuple(q.shape)}, k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} do not fit together")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new must be given together")
    if k_new is not None:
        if _overlaps(k_pages) or _overlaps(v_pages):
            raise ValueError("new rows cannot be written to a broadcast view")
        for t in (k_new, v_new):
            _like(t, q.dtype, (b, k_new.shape[1], hk, d), "k_new / v_new")
    if weights is not None and weights_out is None:
        raise ValueError("weights without weights_out")
    max_pages, cap = _table(block_table, k_pages, b, "block_table")
    _like(seqlens_k, torch.int32, (b,), "seqlens_k")
    o = o or _fresh(q.shape, q.dtype, q.device)
    lse = lse or _fresh((b, h, sq), torch.float32, q.device)
    _like(o, q.dtype, q.shape, "o")
    if _overlaps(o):
        raise ValueError("o must not be a broadcast view")
    _like(lse, torch.float32, (b, h, sq), "lse")
    for t, what in ((weights, "weights"), (weights_out, "weights_out")):
        _like(t, torch.float32, (b, hk, cap), what)
    for t, what in ((weights, "weights"), (weights_out, "weights_out"), (lse, "lse"), (seqlens_k, "seqlens_k")):
        _dense(t, what)
    _on(q.device, k_pages, v_pages, k_new, v_new, block_table, seqlens_k, o, lse, weights, weights_out)
    mode = 0 if weights_out is None else 1 if weights is None else 2
    return _plan("paged", q.dtype, _paged_blob(q, k_pages, v_pages, k_new, v_new, o, scale, window, n_sink, max_pages, mode))


@_on_stream
def flash_attn_paged(q, k_pages, v_pages, block_table, seqlens_k, scale, window=(-1, 0), n_sink=0, k_new=None, v_new=None, weights=None,
                     weights_out=None, out=None, workspace=None):
    """Attention of a few query rows over a key/value cache in pages.  q [b, sq, h, d]; k_pages, v_pages
    [num_pages, page_size, h_k, d]; block_table int32 [b, max_pages]: row j of sequence i is row
    j % page_size of page block_table[i][j // page_size].  block_table None: a dense cache
    [b, capacity, h_k, d].  seqlens_k int32 [b]: rows in the cache before the call; a negative length
    marks an idle sequence (o = 0, lse = +inf, nothing appended).
    k_new, v_new [b, n, h_k, d] are written to the cache IN PLACE at rows seqlens_k[i].. first; rows
    behind the capacity are dropped.  q then attends to rows [0, seqlens_k[i] + n) with the window
    aligned to their end, plus the first n_sink rows (see flash_attn_sink_fwd).  Keys on a page whose
    number lies outside the pool are not seen; rows that no query row sees are not read.  A page
    that receives new rows must appear once, in one sequence's table.
    weights / weights_out f32 [b, h_k, capacity] (weights_out may be weights): when weights_out is given,
    weights_out[i, c, j] = weights[i, c, j] (0 without weights, and for rows appended by this call) + the
    attention that key j got from all query rows and heads of key/value head c, for the rows j in
    the cache after the call; the others are left as they were.  Without query rows (sq 0) new rows are refused.
    -> (o, lse[b, h, sq] f32), and weights_out when given."""
    o, lse = out if out is not None else (None, None)
    scale, n_sink = _nums(scale, n_sink)
    plan = _plan_paged(_sig(q), _sig(k_pages), _sig(v_pages), _sig(block_table), _sig(seqlens_k), _sig(k_new), _sig(v_new), _sig(weights),
                       _sig(weights_out), _sig(o), _sig(lse), scale, _window(window), n_sink)
    if out is None:
        b, sq, h, _ = q.shape
        o, lse = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty((b, h, sq), dtype=torch.float32, device=q.device)
    _launch(plan, _pack11(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_new), _ptr(v_new), _ptr(block_table), seqlens_k.data_ptr(),
                          o.data_ptr(), lse.data_ptr(), _ptr(weights), _ptr(weights_out)), q, workspace)
    return (o, lse) if weights_out is None else (o, lse, weights_out)


def pack_flash_evict_args(k, v, k_out, v_out, b, max_pages, max_pages_out, budget, n_sink, n_recent):
    """The 192-byte extra_args blob of flash_attn_evict, 24 i64: the outer (page), row and head strides of k, v,
    k_out, v_out; b, h_k, d; num_pages, page_size, max_pages of the cache and of the output cache; budget,
    n_sink, n_recent."""
    return _evict_blob(*_sigs(_sig(k), _sig(v), _sig(k_out), _sig(v_out)), b, max_pages, max_pages_out, budget, n_sink, n_recent)


def _evict_blob(k, v, k_out, v_out, b, max_pages, max_pages_out, budget, n_sink, n_recent):
    each = [_strides(t) for t in (k, v, k_out, v_out)]
    return struct.pack("<24q", *[s[i] for i in range(3) for s in each], b, k.shape[2], k.shape[3], k.shape[0], k.shape[1], max_pages,
                       k_out.shape[0], k_out.shape[1], max_pages_out, budget, n_sink, n_recent)


@functools.lru_cache(_PLANS)
def _plan_evict(k, v, weights, seqlens_k, block_table, k_out, v_out, out_table, weights_out, seqlens_out, kept, budget, n_sink, n_recent):
    k, v, weights, seqlens_k, block_table, k_out, v_out, out_table, weights_out, seqlens_out, kept = _sigs(
        k, v, weights, seqlens_k, block_table, k_out, v_out, out_table, weights_out, seqlens_out, kept)
    if (k_out is None) != (v_out is None):
        raise ValueError("k_out and v_out must be given together")
    if budget < 1:
        raise ValueError(f"budget {budget} is not positive")
    _half(k, v, k_out, v_out)
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    b, hk = seqlens_k.shape[0] if len(seqlens_k.shape) == 1 else -1, k.shape[2]
    if k_out is None:
        if out_table is not None:
            raise ValueError("out_table without k_out")
        k_out, v_out, out_table = k, v, block_table
    elif k_out.shape != v_out.shape or k_out.shape[2:] != k.shape[2:]:
        raise ValueError(f"k_out {tuple(k_out.shape)} and v_out {tuple(v_out.shape)} do not fit k {tuple(k.shape)}")
    if _overlaps(k_out) or _overlaps(v_out):
        raise ValueError("rows cannot be moved to a broadcast view")
    max_pages, cap = _table(block_table, k, b, "block_table")
    max_pages_out, cap_out = _table(out_table, k_out, b, "out_table")
    for t, dtype, shape, what in ((seqlens_k, torch.int32, (b,), "seqlens_k"), (seqlens_out, torch.int32, (b,), "seqlens_out"),
                                  (kept, torch.int32, (b, hk, budget), "kept"), (weights, torch.float32, (b, hk, cap), "weights"),
                                  (weights_out, torch.float32, (b, hk, cap_out), "weights_out")):
        _like(t, dtype, shape, what)
        _dense(t, what)
    _on(k.device, v, weights, seqlens_k, block_table, k_out, v_out, out_table, weights_out, seqlens_out, kept)
    return _plan("evict", k.dtype, _evict_blob(k, v, k_out, v_out, b, max_pages, max_pages_out, budget, n_sink, n_recent)) + (cap_out,)


@_on_stream
def flash_attn_evict(k, v, weights, seqlens_k, budget, n_sink=0, n_recent=0, block_table=None, k_out=None, v_out=None, out_table=None,
                     weights_out=None, seqlens_out=None, kept=None):
    """Cuts every (sequence, key/value head) of a cache to `budget` rows: the first n_sink, the last n_recent
    and, of those between, the ones of greatest weight (equal weights: the lower row; NaN below everything)
    stay and move to the front in their order.  k, v: pages with block_table, or dense [b, s, h_k, d];
    weights f32 [b, h_k, capacity] (what flash_attn_paged accumulates); seqlens_k int32 [b].
    Without k_out / v_out the cache, weights and seqlens_k are updated IN PLACE; with them (pages with
    out_table, or dense) the rows that stay are copied there and the cache is left alone.  A sequence of
    at most `budget` rows keeps them all; a negative length stays.  Rows, weights behind the last kept
    one and rows of absent pages are left as they were.  A page that rows move to must appear once, in one
    sequence's table: pages that sequences share (a common prefix) are cut into another cache.
    -> (kept int32 [b, h_k, budget]: the row each came from, -1 behind the last; weights_out; seqlens_out)."""
    plan = _plan_evict(_sig(k), _sig(v), _sig(weights), _sig(seqlens_k), _sig(block_table), _sig(k_out), _sig(v_out), _sig(out_table),
                       _sig(weights_out), _sig(seqlens_out), _sig(kept), *map(operator.index, (budget, n_sink, n_recent)))
    in_place = k_out is None
    b, hk = seqlens_k.shape[0], k.shape[2]
    if in_place:
        k_out, v_out, out_table = k, v, block_table
    if weights_out is None:
        weights_out = weights if in_place else torch.zeros((b, hk, plan[4]), dtype=torch.float32, device=k.device)
    if seqlens_out is None:
        seqlens_out = seqlens_k if in_place else torch.empty_like(seqlens_k)
    if kept is None:
        kept = torch.empty((b, hk, budget), dtype=torch.int32, device=k.device)
    _launch(plan[:4], _pack11(k.data_ptr(), v.data_ptr(), weights.data_ptr(), seqlens_k.data_ptr(), _ptr(block_table), k_out.data_ptr(), v_out.data_ptr(),
                              _ptr(out_table), weights_out.data_ptr(), seqlens_out.data_ptr(), kept.data_ptr()), k, None)
    return kept, weights_out, seqlens_out
