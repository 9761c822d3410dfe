"""Torch-tensor front ends for sf_gemm, sf_rmsnorm, sf_add_rmsnorm,
sf_dequant_int8, sf_gemm_w4 and sf_heads_rope (test and bench plumbing: torch
supplies device memory and the stream; the arithmetic runs in
libsf_hip_kernels.so)."""
from __future__ import annotations

import ctypes
import dataclasses
import struct

import torch

from . import abi

_DT = {torch.bfloat16: abi.SF_BF16, torch.float32: abi.SF_F32, torch.float16: abi.SF_F16, torch.int8: abi.SF_I8}


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _desc(a, w, bias, act, w_scale):
    M, K = a.shape
    d = abi.GemmDesc()
    d.M, d.N, d.K = M, w.shape[0], K
    d.A, d.lda, d.a_dtype = a.data_ptr(), a.stride(0), _DT[a.dtype]
    d.W, d.ldw, d.w_dtype = w.data_ptr(), w.stride(0), _DT[w.dtype]
    d.w_scale = _p(w_scale)
    d.bias = _p(bias)
    d.act = act
    return d


def _run(d, a, workspace):
    """workspace: "auto" allocates what the split-K path needs, None runs the
    single-pass path, a tensor is used as given."""
    if isinstance(workspace, str):
        nbytes = abi.lib().sf_gemm_workspace_bytes(ctypes.byref(d))
        workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=a.device) if nbytes else None
    if workspace is not None:
        d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    abi.check(abi.lib().sf_gemm(ctypes.byref(d), _stream(a)), "sf_gemm")


def workspace_bytes(a, w):
    d = _desc(a, w, None, 0, None)
    return abi.lib().sf_gemm_workspace_bytes(ctypes.byref(d))


def _row_scale(d, row_ss, row_n, row_eps):
    """The activation rows are x * gamma of a deferred RMSNorm with tile sums
    row_ss ([row_n / 64, M] fp32)."""
    if row_ss is not None:
        d.a_row_ss, d.a_row_tiles, d.a_row_n, d.a_row_eps = row_ss.data_ptr(), row_ss.shape[0], row_n, row_eps


def _w16(d, w16):
    """An fp16 copy of the weights (weights_to_f16) for the library path."""
    if w16 is not None:
        d.w_codes16, d.w16_f16 = w16.data_ptr(), 1


def gemm(a, w, bias=None, act=abi.SF_ACT_NONE, out=None, out_dtype=torch.bfloat16,
         accumulate=False, w_scale=None, workspace="auto", w_codes16=None, w16=None, row_ss=None, row_n=0,
         row_eps=1e-6):
    """out[M,N] = act(a[M,K] w[N,K]^T + bias) (bf16 a; bf16 or int8 w with
    per-row fp32 w_scale).  accumulate adds into an fp32 `out`.  w_codes16:
    int8 w's codes as bf16 (int8_codes_to_bf16), read by the library path
    instead of widening them.  w16: an fp16 copy of w (weights_to_f16) for
    fp16 `a`: the library path then multiplies in fp16.  int8 w without a
    copy above 160 rows is read directly when the call fits
    (sf_gemm_int8_direct: K = 2048, N % 256 == 0, fp16 a and out)."""
    M, K = a.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    d = _desc(a, w, bias, act, w_scale)
    d.w_codes16 = _p(w_codes16)
    _w16(d, w16)
    _row_scale(d, row_ss, row_n, row_eps)
    d.epilogue = abi.SF_EPI_PLAIN
    d.C, d.ldc, d.c_dtype = out.data_ptr(), out.stride(0), _DT[out.dtype]
    d.accumulate = 1 if accumulate else 0
    _run(d, a, workspace)
    return out


def gemm_add_norm(a, w, bias, residual, gamma, eps=1e-6, act=abi.SF_ACT_NONE, w_scale=None,
                  norm_dtype=torch.bfloat16, workspace="auto", round_product=False, w16=None, norm_ss=None):
    """residual (fp32 [M,N]) += act(a w^T + bias); returns
    rmsnorm(residual) * gamma in norm_dtype.  round_product: above 160 rows
    the branch output is stored in 16 bits before the add (bf16, or fp16
    with w16)."""
    M = a.shape[0]
    N = w.shape[0]
    out = torch.empty(M, N, dtype=norm_dtype, device=a.device)
    d = _desc(a, w, bias, act, w_scale)
    _w16(d, w16)
    d.epilogue = abi.SF_EPI_ADD_NORM
    d.C, d.ldc, d.c_dtype = residual.data_ptr(), residual.stride(0), abi.SF_F32
    d.eps = eps
    d.norm_gamma, d.norm_out = gamma.data_ptr(), out.data_ptr()
    d.norm_ldo, d.norm_dtype = out.stride(0), _DT[norm_dtype]
    d.round_product = 1 if round_product else 0
    if norm_ss is not None:   # deferred form: out = residual * gamma, tile sums of squares to norm_ss
        d.norm_ss = norm_ss.data_ptr()
    _run(d, a, workspace)
    return out


def gemm_heads(a, w, bias, S, H, outs, gammas=(None, None, None), eps=1e-6, w_scale=None,
               workspace="auto", round_product=False, w16=None, row_ss=None, row_n=0, row_eps=1e-6):
    """Projection whose N columns are sections of H*64, written per head to
    outs[j] ([B,H,S,64] bf16 views) with optional per-head RMSNorm.
    round_product: above 160 rows the projection is stored in 16 bits
    before the norm (bf16, or fp16 with w16 or with int8 w multiplied
    directly, sf_gemm_int8_direct)."""
    d = _desc(a, w, bias, abi.SF_ACT_NONE, w_scale)
    _w16(d, w16)
    _row_scale(d, row_ss, row_n, row_eps)
    d.epilogue = abi.SF_EPI_HEADS
    d.H, d.S, d.eps = H, S, eps
    d.round_product = 1 if round_product else 0
    for j, o in enumerate(outs):
        d.head_out[j] = o.data_ptr()
        d.head_gamma[j] = _p(gammas[j])
        d.head_stride[j][:] = (o.stride(0), o.stride(1), o.stride(2))
    _run(d, a, workspace)
    return outs


def int8_codes_to_bf16(qs):
    """bf16 copies [N][K] of the codes of int8 matrices (row-strided views
    allowed), all in one launch (at most abi.SF_CODES_MAX_JOBS)."""
    outs = [torch.empty(q.shape[0], q.shape[1], dtype=torch.bfloat16, device=q.device) for q in qs]
    jobs = (abi.CodesJob * max(1, len(qs)))()
    for j, (q, o) in enumerate(zip(qs, outs)):
        jobs[j].q, jobs[j].ldq, jobs[j].out = q.data_ptr(), q.stride(0), o.data_ptr()
        jobs[j].N, jobs[j].K = q.shape[0], q.shape[1]
    st = abi.lib().sf_int8_codes_to_bf16(jobs, len(qs), _stream(qs[0]) if qs else None)
    abi.check(st, "sf_int8_codes_to_bf16")
    return outs


def weights_to_f16(ws):
    """fp16 copies [N][K] of bf16 or int8 (codes) matrices, one launch (at
    most abi.SF_CODES_MAX_JOBS)."""
    outs = [torch.empty(w.shape[0], w.shape[1], dtype=torch.float16, device=w.device) for w in ws]
    jobs = (abi.W16Job * max(1, len(ws)))()
    for j, (w, o) in enumerate(zip(ws, outs)):
        jobs[j].w, jobs[j].w_dtype, jobs[j].ldw = w.data_ptr(), _DT[w.dtype], w.stride(0)
        jobs[j].out, jobs[j].N, jobs[j].K = o.data_ptr(), w.shape[0], w.shape[1]
    abi.check(abi.lib().sf_weights_to_f16(jobs, len(ws), _stream(ws[0]) if ws else None), "sf_weights_to_f16")
    return outs


def frag_pack(ws, out_dtypes):
    """Fragment-ordered copies (sf_frag_pack) of row-major matrices, one
    launch (at most abi.SF_CODES_MAX_JOBS)."""
    outs = [torch.empty(w.shape[0], w.shape[1], dtype=dt, device=w.device) for w, dt in zip(ws, out_dtypes)]
    jobs = (abi.FragJob * max(1, len(ws)))()
    for j, (w, o) in enumerate(zip(ws, outs)):
        jobs[j].w, jobs[j].w_dtype, jobs[j].ldw = w.data_ptr(), _DT[w.dtype], w.stride(0)
        jobs[j].out, jobs[j].out_dtype, jobs[j].N, jobs[j].K = o.data_ptr(), _DT[o.dtype], w.shape[0], w.shape[1]
    abi.check(abi.lib().sf_frag_pack(jobs, len(ws), _stream(ws[0]) if ws else None), "sf_frag_pack")
    return outs


def _frag_desc(M, a, w, bias, act, w_scale, row_ss, row_n, row_eps):
    d = abi.FragGemmDesc()
    d.M, d.N, d.K = M, w.shape[0], w.shape[1]
    d.A, d.a_dtype = a.data_ptr(), _DT[a.dtype]
    d.W, d.w_dtype = w.data_ptr(), _DT[w.dtype]
    d.w_scale, d.bias, d.act = _p(w_scale), _p(bias), act
    if row_ss is not None:
        d.a_row_ss, d.a_row_tiles, d.a_row_n, d.a_row_eps = row_ss.data_ptr(), row_ss.shape[1], row_n, row_eps
    return d


def _run_frag(d, t):
    abi.check(abi.lib().sf_gemm_frag(ctypes.byref(d), _stream(t)), "sf_gemm_frag")


def gemm_frag(M, a, w, bias=None, act=abi.SF_ACT_NONE, out=None, out_dtype=torch.float32, c_frag=False,
              accumulate=False, w_scale=None, row_ss=None, row_n=0, row_eps=1e-6, x=None, x_gamma=None):
    """sf_gemm_frag's plain epilogue on M rows of a (fragment order, padded
    rows) and w (frag_pack): row-major [M, N], or fragment order with c_frag.
    x, x_gamma: the fp32 rows and gamma behind deferred fp16 rows (required)."""
    N = w.shape[0]
    d = _frag_desc(M, a, w, bias, act, w_scale, row_ss, row_n, row_eps)
    if out is None:
        out = torch.empty((M + 15) // 16 * 16 if c_frag else M, N, dtype=out_dtype, device=a.device)
    d.epilogue = abi.SF_EPI_PLAIN
    d.C, d.ldc, d.c_dtype = out.data_ptr(), N if c_frag else out.stride(0), _DT[out.dtype]
    d.c_frag, d.accumulate = int(c_frag), int(accumulate)
    if x is not None:
        d.a_x, d.a_x_ld, d.a_x_gamma = x.data_ptr(), x.stride(0), x_gamma.data_ptr()
    _run_frag(d, a)
    return out


def gemm_frag_heads(M, a, w, bias, S, H, outs, gammas=(None, None, None), eps=1e-6, w_scale=None, row_ss=None,
                    row_n=0, row_eps=1e-6):
    """sf_gemm_frag's per-head epilogue (outs: [B,H,S,64] bf16 views)."""
    d = _frag_desc(M, a, w, bias, abi.SF_ACT_NONE, w_scale, row_ss, row_n, row_eps)
    d.epilogue, d.H, d.S, d.eps = abi.SF_EPI_HEADS, H, S, eps
    for j, o in enumerate(outs):
        d.head_out[j], d.head_gamma[j] = o.data_ptr(), _p(gammas[j])
        d.head_stride[j][:] = (o.stride(0), o.stride(1), o.stride(2))
    _run_frag(d, a)
    return outs


def gemm_frag_add_norm(M, a, w, bias, residual, gamma, norm_dtype=torch.bfloat16, w_scale=None):
    """sf_gemm_frag's residual add + deferred RMSNorm: residual (fp32 [M, N])
    += a w^T + bias; returns (residual * gamma in fragment order, tile sums
    of squares)."""
    N = w.shape[0]
    d = _frag_desc(M, a, w, bias, abi.SF_ACT_NONE, w_scale, None, 0, 0.0)
    out = torch.empty((M + 15) // 16 * 16, N, dtype=norm_dtype, device=a.device)
    ss = torch.empty(M, abi.lib().sf_gemm_frag_ss_tiles(ctypes.byref(d)), dtype=torch.float32, device=a.device)
    d.epilogue = abi.SF_EPI_ADD_NORM
    d.C, d.ldc, d.c_dtype = residual.data_ptr(), residual.stride(0), abi.SF_F32
    d.norm_gamma, d.norm_out, d.norm_dtype, d.norm_ss = gamma.data_ptr(), out.data_ptr(), _DT[norm_dtype], ss.data_ptr()
    _run_frag(d, a)
    return out, ss


def norm_frag(x, gamma, eps=1e-6, out_dtype=torch.bfloat16, deferred=False):
    """sf_norm_frag on fp32 rows: (fragment-ordered norm or x * gamma, tile
    sums or None)."""
    rows, cols = x.shape
    out = torch.empty((rows + 15) // 16 * 16, cols, dtype=out_dtype, device=x.device)
    ss = torch.empty(rows, cols // 64, dtype=torch.float32, device=x.device) if deferred else None
    st = abi.lib().sf_norm_frag(x.data_ptr(), x.stride(0), gamma.data_ptr(), out.data_ptr(), _DT[out_dtype], _p(ss),
                                rows, cols, eps, _stream(x))
    abi.check(st, "sf_norm_frag")
    return out, ss


def rmsnorm_deferred(x, gamma, out_dtype=torch.bfloat16):
    """sf_rmsnorm_deferred on fp32 rows x [rows, cols]: (x * gamma in
    out_dtype, tile sums of squares [cols / 64, rows] fp32)."""
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=out_dtype, device=x.device)
    ss = torch.empty(cols // 64, rows, dtype=torch.float32, device=x.device)
    st = abi.lib().sf_rmsnorm_deferred(x.data_ptr(), x.stride(0), gamma.data_ptr(), out.data_ptr(), _DT[out_dtype],
                                       out.stride(0), ss.data_ptr(), rows, cols, _stream(x))
    abi.check(st, "sf_rmsnorm_deferred")
    return out, ss


def rmsnorm(x, gamma, eps=1e-6, out_dtype=torch.bfloat16, out=None):
    rows, cols = x.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=out_dtype, device=x.device)
    st = abi.lib().sf_rmsnorm(x.data_ptr(), _DT[x.dtype], x.stride(0), gamma.data_ptr(),
                              out.data_ptr(), _DT[out.dtype], out.stride(0), rows, cols, eps,
                              _stream(x))
    abi.check(st, "sf_rmsnorm")
    return out


def add_rmsnorm(delta, residual, gamma, eps=1e-6, out_dtype=torch.bfloat16):
    rows, cols = residual.shape
    out = torch.empty(rows, cols, dtype=out_dtype, device=residual.device)
    st = abi.lib().sf_add_rmsnorm(delta.data_ptr(), _DT[delta.dtype], residual.data_ptr(),
                                  gamma.data_ptr(), out.data_ptr(), _DT[out.dtype], rows, cols,
                                  eps, _stream(residual))
    abi.check(st, "sf_add_rmsnorm")
    return out


def dequant_int8(q, scale, per_channel=True, out_dtype=torch.float32):
    N = q.shape[0]
    K = q.numel() // max(N, 1)
    out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    st = abi.lib().sf_dequant_int8(q.data_ptr(), scale.data_ptr(), 1 if per_channel else 0,
                                   out.data_ptr(), _DT[out_dtype], N, K, _stream(q))
    abi.check(st, "sf_dequant_int8")
    return out


def _raw_stream(device):
    """The raw handle of torch's current stream on `device`, without building a Stream object (2 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def call_on(device, what, fn, *args):
    """fn(*args, stream) on torch's current stream of `device`, with that device current (kernels are loaded and
    launched on the current one); raises on an error status."""
    if device.index == torch.cuda.current_device():
        st = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _raw_stream(device))
    if st:
        abi.check(st, what)


_B16 = (torch.bfloat16, torch.float16)
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _check(t, name, dtypes, device=None, dim=None):
    """t is a device tensor of one of dtypes (on `device`, with dim axes and a contiguous last one)."""
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be a device tensor" + ("" if device is None else f" on {device}"))
    if t.dtype not in dtypes:
        raise ValueError(f"{name} is {t.dtype}: {' or '.join(str(d) for d in dtypes)} expected")
    if dim is not None and (t.dim() != dim or (t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel())):
        raise ValueError(f"{name}{tuple(t.shape)}: {dim} axes with a contiguous last one expected")


def _vector(t, name, dtype, n, device):
    """The pointer of a contiguous device tensor of n elements (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.device != device or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}{tuple(t.shape)} {t.dtype}: {n} contiguous {dtype} on {device} expected")
    return t.data_ptr()


def strides_bhs(t):
    """Element strides of [B, H, S, D], 0 for an axis of one (torch leaves any number there)."""
    n, st = t.shape, t.stride()
    return (st[0] if n[0] > 1 else 0, st[1] if n[1] > 1 else 0, st[2] if n[2] > 1 else 0)


@dataclasses.dataclass(frozen=True)
class W4:
    """4-bit weights [N, K] as sf_gemm_w4 reads them (w4_pack)."""

    data: torch.Tensor
    N: int
    K: int
    group: int
    scale_dtype: torch.dtype


def w4_pack(codes, scales, zeros=None, group=128):
    """Lays 4-bit weights out once for gemm_w4.  codes: uint8 [N, K / 2], input
    2 i of a row in the low half of byte i, 2 i + 1 in the high half; scales:
    fp16 or bf16 [N, K / group]; zeros: uint8 [N, K / group] or None (8).  The
    weight is scale * (code - zero)."""
    _check(codes, "codes", (torch.uint8,), dim=2)
    dev, (N, half) = codes.device, codes.shape
    K = 2 * half
    need = abi.lib().sf_w4_bytes(N, K, group)
    if need == 0:
        raise ValueError(f"no 4-bit weights [{N}, {K}] in groups of {group}: 32, 64 or 128, K a multiple")
    _check(scales, "scales", _B16, dev, 2)
    if zeros is not None:
        _check(zeros, "zeros", (torch.uint8,), dev, 2)
    for name, t in (("scales", scales), ("zeros", zeros)):
        if t is not None and t.shape != (N, K // group):
            raise ValueError(f"{name}{tuple(t.shape)}: [{N}, {K // group}] expected")
    d = abi.W4PackDesc()
    d.N, d.K, d.group = N, K, group
    d.codes, d.ldc = codes.data_ptr(), codes.stride(0) if N > 1 else half
    d.scales, d.lds, d.scale_dtype = scales.data_ptr(), scales.stride(0) if N > 1 else K, _DT[scales.dtype]
    if zeros is not None:
        d.zeros, d.ldz = zeros.data_ptr(), zeros.stride(0) if N > 1 else K
    out = torch.empty(need, dtype=torch.uint8, device=dev)
    call_on(dev, "sf_w4_pack", abi.lib().sf_w4_pack, ctypes.byref(d), out.data_ptr())
    return W4(out, N, K, group, scales.dtype)


def gemm_w4(a, w, bias=None, act=abi.SF_ACT_NONE, out=None, out_dtype=None, accumulate=False):
    """out[M, N] = act(a[M, K] W^T + bias) with 4-bit weights w (w4_pack); a
    bf16 or fp16, out_dtype a's unless given.  accumulate adds into an fp32
    `out`."""
    dev, N, K = w.data.device, w.N, w.K
    _check(a, "a", _B16, dev, 2)
    M = a.shape[0]
    if a.shape[1] != K:
        raise ValueError(f"a{tuple(a.shape)} against weights [{N}, {K}]")
    if out is None:
        if accumulate:
            raise ValueError("accumulate adds into out: give one")
        out = torch.empty(M, N, dtype=out_dtype or a.dtype, device=dev)
    else:
        _check(out, "out", _FLOATS, dev, 2)
        if out.shape != (M, N) or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out{tuple(out.shape)} {out.dtype}: [{M}, {N}] of {out_dtype or out.dtype} expected")
    d = abi.GemmW4Desc(M, N, K, w.group, a.data_ptr(), a.stride(0) if M > 1 else K, _DT[a.dtype], w.data.data_ptr(),
                       _DT[w.scale_dtype], _vector(bias, "bias", torch.float32, N, dev), act, out.data_ptr(),
                       out.stride(0) if M > 1 else N, _DT[out.dtype], 1 if accumulate else 0)
    call_on(dev, "sf_gemm_w4", abi.lib().sf_gemm_w4, ctypes.byref(d))
    return out


# sf_heads_rope_desc in one pack (a ctypes structure of nested arrays takes 3 us to fill).
_ROPE_DESC = struct.Struct("@8i3P9q3P9q2Pf4x2P2iP4iP")
assert _ROPE_DESC.size == ctypes.sizeof(abi.HeadsRopeDesc)
_NO_CACHE = (0, 0, 0, 0, 0)


def _heads_rope(dev, n, head, src, src_st, out, out_st, D, gammas, positions, inv_freq, interleaved, eps, cache, slots):
    """The call: head = (B, S, D, Hq, Hk, Hv, in_dtype, out_dtype), pointers and strides flat, n = B * S tokens."""
    gq, gk = gammas
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    if cache is not None and cache.data.device != dev:
        raise ValueError(f"the cache must be on {dev}")
    raw = _ROPE_DESC.pack(
        *head, *src, *src_st, *out, *out_st, _vector(gq, "gamma", torch.float32, D, dev),
        _vector(gk, "gamma", torch.float32, D, dev), eps, _vector(positions, "positions", torch.int32, n, dev),
        _vector(inv_freq, "inv_freq", torch.float64, rot // 2, dev), rot, 1 if interleaved else 0,
        *(_NO_CACHE if cache is None else cache.fields()), _vector(slots, "slots", torch.int32, n, dev))
    call_on(dev, "sf_heads_rope", abi.lib().sf_heads_rope, ctypes.byref(abi.HeadsRopeDesc.from_buffer_copy(raw)))


def heads_rope_strided(srcs, outs, gammas=(None, None), positions=None, inv_freq=None, interleaved=False, eps=1e-6,
                       cache=None, slots=None):
    """sf_heads_rope on query, key and value views [B, heads, S, D] (None: left
    out), written to outs (views of the same shapes; key and value None with a
    cache, attention.Kv4Cache)."""
    like = next((t for t in srcs if t is not None), None)
    if like is None or len(srcs) != 3 or len(outs) != 3:
        raise ValueError("three sources and outputs, query, key and value, not all of them None")
    _check(like, "source", _FLOATS, None, 4)
    dev, (B, _, S, D) = like.device, like.shape
    heads, src, src_st, out, out_st, out_dtype = [0, 0, 0], [0, 0, 0], [], [0, 0, 0], [], None
    for j, (t, o) in enumerate(zip(srcs, outs)):
        if (o is None) != (t is None or (cache is not None and j > 0)):
            raise ValueError("an output for every source; none for keys and values that go into a cache")
        if t is not None:
            _check(t, "source", (like.dtype,), dev, 4)
            if (t.shape[0], t.shape[2], t.shape[3]) != (B, S, D):
                raise ValueError(f"source {tuple(t.shape)} beside {tuple(like.shape)}")
            heads[j], src[j] = t.shape[1], t.data_ptr()
        if o is not None:
            out_dtype = out_dtype or o.dtype
            _check(o, "output", (out_dtype,) if out_dtype in _FLOATS else _FLOATS, dev, 4)
            if o.shape != t.shape:
                raise ValueError(f"output {tuple(o.shape)} for a source {tuple(t.shape)}")
            out[j] = o.data_ptr()
        src_st += (0, 0, 0) if t is None else strides_bhs(t)
        out_st += (0, 0, 0) if o is None else strides_bhs(o)
    _heads_rope(dev, B * S, (B, S, D, *heads, _DT[like.dtype], _DT[out_dtype or like.dtype]), src, src_st, out, out_st, D,
                gammas, positions, inv_freq, interleaved, eps, cache, slots)


def heads_rope(p, S, heads, D, gammas=(None, None), positions=None, inv_freq=None, interleaved=False, eps=1e-6,
               out_dtype=None, cache=None, slots=None):
    """Splits a projection's rows p [B * S, (Hq + Hk + Hv) * D] into query, key
    and value heads [B, heads, S, D] (heads = (Hq, Hk, Hv), 0 leaves one out),
    with the RMSNorm of each query and key head (gammas, fp32 [D] or None) and
    the rotation of their first 2 * len(inv_freq) channels by the token's
    position (positions: int32 [B * S]; inv_freq: float64 radians a position;
    pairs (i, i + half), or (2 i, 2 i + 1) with interleaved).  A token with a
    negative position is padding and is not written.  With a cache
    (attention.Kv4Cache) keys and values go there, at `slots` (int32) or the
    positions.  Returns (q, k, v), None for what is left out or cached."""
    _check(p, "p", _FLOATS, None, 2)
    dev, (n, cols) = p.device, p.shape
    Hq, Hk, Hv = heads
    if min(heads) < 0 or cols != (Hq + Hk + Hv) * D or S <= 0 or n % S:
        raise ValueError(f"p{tuple(p.shape)}: rows of {sum(heads)} x {D} for tokens in groups of {S} expected")
    B, ld, base, dtype = n // S, p.stride(0) if n > 1 else 0, p.data_ptr(), out_dtype or p.dtype
    step = D * p.element_size()
    q, k, v = (torch.empty(B, h, S, D, dtype=dtype, device=dev) if h and (cache is None or j == 0) else None
               for j, h in enumerate(heads))
    _heads_rope(dev, n, (B, S, D, Hq, Hk, Hv, _DT[p.dtype], _DT[dtype]),
                (base, base + Hq * step, base + (Hq + Hk) * step), (S * ld, D, ld) * 3,
                tuple(0 if t is None else t.data_ptr() for t in (q, k, v)),
                (Hq * S * D, S * D, D, Hk * S * D, S * D, D, Hv * S * D, S * D, D),
                D, gammas, positions, inv_freq, interleaved, eps, cache, slots)
    return q, k, v
