"""Operator layer with the names and argument lists of the reference's compiled
module ``superl8._C`` (reference csrc/fni8_api.cpp:225-291), implemented over the
C ABI of ``libsuperl8_b200.so``.

Each function validates like the reference's ``TORCH_CHECK``s (same key words in
the messages), allocates outputs/workspaces with torch on the inputs' device and
launches on torch's current stream.  Nothing here computes on the CPU.
"""

from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

# Two bindings serve the reference's six compiled operators (quantize_i8_rowwise, attn_int8_fwd,
# attn_int8_fwd_train, attn_fp16_fwd, attn_bwd, attn_int8_decode): the compiled torch extension
# ``_C_ext`` (csrc/torch_ext, built by ``python -m superl8_b200.build``) when it is present, and
# ctypes otherwise.  Both end in the same C-ABI calls.  Calls that use an argument the reference's
# operators do not have (seqlens, backend, out, gate_flag, context_lens) always take ctypes.
try:
    from . import _C_ext as _ext
except ImportError:          # not built: the ctypes binding serves everything
    _ext = None
BINDING = "compiled" if _ext is not None else "ctypes"


def use_binding(name: str) -> str:
    """Selects "compiled" or "ctypes" for the six reference operators; returns the previous choice."""
    global BINDING
    if name not in ("compiled", "ctypes"):
        raise ValueError(name)
    if name == "compiled" and _ext is None:
        raise RuntimeError("superl8_b200: the compiled extension _C_ext is not built (python -m superl8_b200.build)")
    prev, BINDING = BINDING, name
    return prev


def _compiled() -> bool:
    return BINDING == "compiled"


_DTYPE = {torch.float16: _lib.SL8_F16, torch.bfloat16: _lib.SL8_BF16, torch.float32: _lib.SL8_F32}
_status_ws: dict = {}
_decode_ws: dict = {}
_bwd_ws: dict = {}      # the last backward workspace per (device, stream): its status word is read by device_status


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _status_buffer(device) -> torch.Tensor:
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    buf = _status_ws.get(key)
    if buf is None:
        buf = torch.zeros(64, dtype=torch.int32, device=device)
        _status_ws[key] = buf
    return buf


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _check_cuda(*ts) -> None:
    _check(all(t.is_cuda for t in ts), "superl8_b200: all inputs (incl. scales) must be CUDA tensors")
    _check(all(t.device == ts[0].device for t in ts), "superl8_b200: all inputs must be on the same device")


def device_status(device=None) -> int:
    """Synchronises and returns the device status word of the current stream's
    status buffer (0, or the DEVICE_TIMEOUT code when a bounded wait expired)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    lib = _lib.load()
    rc = lib.sl8_read_device_status(_ptr(_status_buffer(device)), _stream(device))
    ws = _decode_ws.get((device.index, torch.cuda.current_stream(device).cuda_stream))
    if rc == 0 and ws is not None:
        rc = lib.sl8_read_device_status(_ptr(ws), _stream(device))
    bws = _bwd_ws.get((device.index, torch.cuda.current_stream(device).cuda_stream))
    if rc == 0 and bws is not None:
        rc = lib.sl8_read_device_status(_ptr(bws), _stream(device))
    if rc == 0 and _ext is not None:
        rc = int(_ext.device_status(torch.empty(0, device=device)))
    if rc == 0:
        with torch.cuda.device(device):
            rc = lib.sl8_paged_status(_stream(device))
    return rc


def quantize_i8_rowwise(x: torch.Tensor):
    """x [M, K] fp16/bf16/fp32 -> (q int8 [M, K], scale fp32 [M]).
    Reference binding: csrc/fni8_api.cpp:286-291; op csrc/kernel/quant_rowwise.cu:84-121."""
    if _compiled():
        r = _ext.quantize_i8_rowwise(x)
        _lib.launches += 1 if x.numel() else 0
        return r
    _check(x.is_cuda, "superl8_b200 quantize_i8_rowwise: x must be a CUDA tensor")
    _check(x.dim() == 2, "superl8_b200 quantize_i8_rowwise: expect [M, K]")
    _check(x.dtype in _DTYPE, "superl8_b200 quantize_i8_rowwise: x must be float16, bfloat16 or float32")
    x = x.contiguous()
    M, K = x.shape
    q = torch.empty((M, K), dtype=torch.int8, device=x.device)
    scale = torch.empty((M,), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        rc = _lib.load().sl8_quantize_i8_rowwise(_ptr(x), _DTYPE[x.dtype], M, K, _ptr(q), _ptr(scale), _stream(x.device))
    _lib.check(rc, "quantize_i8_rowwise", 1)
    return q, scale


def _fwd_checks(q, q_scale, k, k_scale, v, what):
    _check_cuda(q, q_scale, k, k_scale, v)
    _check(q.dtype == torch.int8 and k.dtype == torch.int8, f"{what}: q/k must be int8")
    _check(q_scale.dtype == torch.float32 and k_scale.dtype == torch.float32, f"{what}: scales must be float32")
    _check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, f"{what}: expect [B,H,S,D]")
    _check(all(t.is_contiguous() for t in (q, q_scale, k, k_scale, v)), f"{what}: inputs must be contiguous")
    B, H, M, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    _check(k.shape[0] == B and v.shape[0] == B and v.shape[1] == Hkv, f"{what}: batch/head mismatch")
    _check(Hkv > 0 and H % Hkv == 0, f"{what}: H_q must be divisible by H_kv (GQA)")
    _check(k.shape[3] == D and v.shape[3] == D and v.shape[2] == N, f"{what}: K/V shape mismatch")
    _check(q_scale.numel() == B * H * M and k_scale.numel() == B * Hkv * N, f"{what}: scale shape mismatch")
    return B, H, Hkv, M, N, D


def _gate_args(gate_flag, gate_want, device, what):
    if gate_flag is None:
        return dict(gate_flag=None, gate_want=0)
    _check(gate_flag.is_cuda and gate_flag.device == device and gate_flag.dtype == torch.int32 and gate_flag.numel() >= 1,
           f"{what}: gate_flag must be an int32 CUDA tensor on the inputs' device")
    return dict(gate_flag=gate_flag.data_ptr(), gate_want=int(bool(gate_want)))


def _run_fwd(q, q_scale, k, k_scale, v, causal, want_lse, window_left, seqlens_q=None, seqlens_k=None,
             backend=_lib.SL8_BACKEND_AUTO, out=None, gate_flag=None, gate_want=False):
    what = "superl8_b200"
    B, H, Hkv, M, N, D = _fwd_checks(q, q_scale, k, k_scale, v, what)
    _check(v.dtype in (torch.float16, torch.bfloat16), f"{what}: v must be float16 or bfloat16")
    _check(D in (32, 64, 72, 80, 128, 256), f"{what}: head dim must be 32/64/72/80/128/256, got {D}")
    if out is None:
        out = torch.empty((B, H, M, D), dtype=v.dtype, device=v.device)
    else:
        _check(out.shape == (B, H, M, D) and out.dtype == v.dtype and out.device == v.device and out.is_contiguous(),
               f"{what}: out must be a contiguous [B,H,M,D] tensor of v's dtype on v's device")
    lse = torch.empty((B, H, M) if want_lse else (0,), dtype=torch.float32, device=q.device)
    if M == 0 or B == 0 or H == 0:
        return out, lse
    for s in (seqlens_q, seqlens_k):
        if s is not None:
            _check(s.is_cuda and s.dtype == torch.int32 and s.numel() == B and s.is_contiguous(),
                   f"{what}: seqlens must be contiguous int32 [B] CUDA tensors")
    p = _lib.FwdParams(
        q=q.data_ptr(), q_scale=q_scale.data_ptr(), k=k.data_ptr(), k_scale=k_scale.data_ptr(), v=v.data_ptr(),
        out=out.data_ptr(), lse=lse.data_ptr() if want_lse else None,
        seqlens_q=None if seqlens_q is None else seqlens_q.data_ptr(),
        seqlens_k=None if seqlens_k is None else seqlens_k.data_ptr(),
        B=B, Hq=H, Hkv=Hkv, M=M, N=N, D=D, v_dtype=_DTYPE[v.dtype], causal=int(bool(causal)),
        window_left=int(window_left), backend=int(backend), **_gate_args(gate_flag, gate_want, q.device, what))
    with torch.cuda.device(q.device):
        ws = _status_buffer(q.device)
        rc = _lib.load().sl8_attn_int8_fwd(C.byref(p), _ptr(ws), ws.numel() * 4, _stream(q.device))
    _lib.check(rc, "attn_int8_fwd", 1)
    return out, lse


def attn_int8_fwd(q, q_scale, k, k_scale, v, causal=False, window_left=-1, *, seqlens_q=None, seqlens_k=None,
                  backend=_lib.SL8_BACKEND_AUTO, out=None, gate_flag=None, gate_want=False):
    """Reference binding csrc/fni8_api.cpp:225-229 (op csrc/kernel/attn_int8_fwd.cu:185-190).
    ``out`` (optional) receives the result; ``gate_flag`` (int32 CUDA tensor, optional) makes the
    launch conditional on the device: the kernel works only if (flag != 0) == gate_want."""
    if (_compiled() and seqlens_q is None and seqlens_k is None and backend == _lib.SL8_BACKEND_AUTO and out is None
            and gate_flag is None):
        r = _ext.attn_int8_fwd(q, q_scale, k, k_scale, v, bool(causal), int(window_left))
        _lib.launches += 1 if r.numel() else 0
        return r
    return _run_fwd(q, q_scale, k, k_scale, v, causal, False, window_left, seqlens_q, seqlens_k, backend,
                    out, gate_flag, gate_want)[0]


def attn_int8_fwd_train(q, q_scale, k, k_scale, v, causal=False, *, backend=_lib.SL8_BACKEND_AUTO):
    """Also returns the natural-log LSE.  Reference binding csrc/fni8_api.cpp:230-233."""
    if _compiled() and backend == _lib.SL8_BACKEND_AUTO:
        r = _ext.attn_int8_fwd_train(q, q_scale, k, k_scale, v, bool(causal))
        _lib.launches += 1 if r[0].numel() else 0
        return r
    return _run_fwd(q, q_scale, k, k_scale, v, causal, True, -1, None, None, backend)


def attn_int8_fwd_fused(q, k, v, causal=False, scale=None, window_left=-1, *, seqlens_q=None, seqlens_k=None,
                        gate=True, ratio_threshold=12.0):
    """attn_int8_fwd from 16-bit q, k, v [B, H, S, D] in ONE library call (sl8_attn_int8_fwd_fused):
    gate, Q / K prologue and both candidate kernels queued back to back, the gate decided on the
    device.  Returns (out, flag): flag is an int32 [1] device tensor, non-zero when the
    full-precision kernel produced ``out``.  D in {64, 128, 256}, one dtype, N > 0."""
    what = "superl8_b200 fused fwd"
    _check_cuda(q, k, v)
    _check(q.dtype in (torch.float16, torch.bfloat16), f"{what}: q must be float16 or bfloat16")
    _check(k.dtype == q.dtype and v.dtype == q.dtype, f"{what}: q, k, v must share one dtype")
    _check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, f"{what}: expect [B,H,S,D]")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    B, H, M, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    _check(k.shape[0] == B and v.shape[0] == B and v.shape[1] == Hkv, f"{what}: batch/head mismatch")
    _check(Hkv > 0 and H % Hkv == 0, f"{what}: H_q must be divisible by H_kv (GQA)")
    _check(k.shape[3] == D and v.shape[3] == D and v.shape[2] == N, f"{what}: K/V shape mismatch")
    _check(D in (64, 128, 256), f"{what}: head dim must be 64/128/256, got {D}")
    for s_ in (seqlens_q, seqlens_k):
        if s_ is not None:
            _check(s_.is_cuda and s_.dtype == torch.int32 and s_.numel() == B and s_.is_contiguous(),
                   f"{what}: seqlens must be contiguous int32 [B] CUDA tensors")
    out = torch.empty((B, H, M, D), dtype=v.dtype, device=v.device)
    sc = (1.0 / math.sqrt(D)) if scale is None else float(scale)
    status = _status_buffer(q.device)      # the stream's shared status word: device_status() reads it
    flag = torch.empty(1, dtype=torch.int32, device=q.device)   # zeroed by the call; outlives the workspace
    p = _lib.FusedFwdParams(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), device_status=status.data_ptr(),
        gate_flag=flag.data_ptr(),
        seqlens_q=None if seqlens_q is None else seqlens_q.data_ptr(),
        seqlens_k=None if seqlens_k is None else seqlens_k.data_ptr(),
        B=B, Hq=H, Hkv=Hkv, M=M, N=N, D=D, dtype=_DTYPE[q.dtype], causal=int(bool(causal)),
        window_left=int(window_left), ratio_threshold=float(ratio_threshold) if gate else 0.0, softmax_scale=sc)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        nbytes = int(lib.sl8_attn_int8_fwd_fused_workspace(C.byref(p)))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rc = lib.sl8_attn_int8_fwd_fused(C.byref(p), _ptr(ws), nbytes, _stream(q.device))
    _lib.check(rc, "attn_int8_fwd_fused",
               (2 + _lib.k_prologue_launches(_DTYPE[k.dtype], B * Hkv, N, D) + (1 if gate else 0)) if out.numel() else 0)
    return out, flag


def qk_logits_i32(q_i8: torch.Tensor, k_i8: torch.Tensor) -> torch.Tensor:
    """int32 q[M,D] . k[N,D]^T on the tcgen05 kind::i8 tile path (no reference op; see the header)."""
    _check(q_i8.is_cuda and k_i8.is_cuda and q_i8.dtype == torch.int8 and k_i8.dtype == torch.int8,
           "superl8_b200 qk_logits_i32: q/k must be int8 CUDA tensors")
    _check(q_i8.dim() == 2 and k_i8.dim() == 2 and q_i8.shape[1] == k_i8.shape[1], "superl8_b200 qk_logits_i32: expect [M,D],[N,D]")
    q_i8, k_i8 = q_i8.contiguous(), k_i8.contiguous()
    M, D = q_i8.shape
    N = k_i8.shape[0]
    _check(D in (64, 128, 256), f"superl8_b200 qk_logits_i32: head dim must be 64/128/256, got {D}")
    s = torch.empty((M, N), dtype=torch.int32, device=q_i8.device)
    with torch.cuda.device(q_i8.device):
        ws = _status_buffer(q_i8.device)
        rc = _lib.load().sl8_qk_logits_i32(_ptr(q_i8), _ptr(k_i8), M, N, D, _ptr(s), _ptr(ws), ws.numel() * 4,
                                           _stream(q_i8.device))
    _lib.check(rc, "qk_logits_i32", 1)
    return s


def tensor_peak(kind_i8: bool, iters: int = 4096, device=None, n_cols: int = 256) -> float:
    """Measured tensor-pipe peak in T(FL)OP/s for kind::i8 (or kind::f16): times the probe launch
    with CUDA events after one warm-up launch.  ``n_cols`` (64, 128, 256) = N of the instruction."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    lib = _lib.load()
    ops = C.c_double(0.0)
    with torch.cuda.device(device):
        ws = _status_buffer(device)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for i in range(2):
            if i == 1:
                e0.record()
            rc = lib.sl8_tensor_peak_probe_n(int(bool(kind_i8)), int(n_cols), int(iters), C.byref(ops), _ptr(ws),
                                             ws.numel() * 4, _stream(device))
            _lib.check(rc, "tensor_peak_probe", 1)
        e1.record()
        torch.cuda.synchronize(device)
    return ops.value / (e0.elapsed_time(e1) * 1e-3) / 1e12


def attn_fp16_fwd(q, k, v, causal=False, scale=None, window_left=-1, mask=None, *, seqlens_q=None, seqlens_k=None,
                  backend=_lib.SL8_BACKEND_AUTO, want_lse=False, out=None, gate_flag=None, gate_want=False):
    """Full-precision forward.  Reference binding csrc/fni8_api.cpp:234-244.  ``want_lse``: also
    return the natural-log row sums [B, H, M] (what the backward consumes).  ``out`` / ``gate_flag`` /
    ``gate_want``: as in attn_int8_fwd (conditional launch decided on the device)."""
    what = "superl8_b200 fp16 fwd"
    if (_compiled() and seqlens_q is None and seqlens_k is None and backend == _lib.SL8_BACKEND_AUTO and out is None
            and gate_flag is None):
        sc_ = None if scale is None else float(scale)
        if want_lse and mask is None and window_left < 0:
            r = _ext.attn_fp16_fwd_train(q, k, v, bool(causal), sc_)
            _lib.launches += 1 if r[0].numel() else 0
            return r
        if not want_lse:
            r = _ext.attn_fp16_fwd(q, k, v, bool(causal), sc_, int(window_left), mask)
            _lib.launches += 1 if r.numel() else 0
            return r
    _check_cuda(q, k, v)
    _check(q.dtype in (torch.float16, torch.bfloat16), f"{what}: q must be float16 or bfloat16")
    _check(k.dtype == q.dtype and v.dtype == q.dtype, f"{what}: q, k, v must share one dtype")
    _check(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, f"{what}: expect [B,H,S,D]")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    B, H, M, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    mk = dict(mask=None, mask_stride_b=0, mask_stride_h=0, mask_stride_m=0, mask_stride_n=0)
    if mask is not None:
        _check(mask.is_cuda and mask.device == q.device, f"{what}: mask must be a CUDA tensor on q's device")
        _check(mask.dtype == q.dtype, f"{what}: mask dtype must match q/k/v")
        _check(mask.dim() == 4, f"{what}: mask must be 4-D [B|1, H|1, M, N]")
        _check(mask.shape[2] == M and mask.shape[3] == N, f"{what}: mask trailing dims must be [M,N]")
        _check(mask.shape[0] in (B, 1) and mask.shape[1] in (H, 1), f"{what}: mask leading dims must broadcast to [B,H]")
        # indexed in place: a broadcast [B,1,M,N] view is never expanded (zero stride on size-1 axes)
        mk = dict(mask=mask.data_ptr(), mask_stride_b=0 if mask.shape[0] == 1 else mask.stride(0),
                  mask_stride_h=0 if mask.shape[1] == 1 else mask.stride(1),
                  mask_stride_m=mask.stride(2), mask_stride_n=mask.stride(3))
    _check(k.shape[0] == B and v.shape[0] == B and v.shape[1] == Hkv, f"{what}: batch/head mismatch")
    _check(Hkv > 0 and H % Hkv == 0, f"{what}: H_q must be divisible by H_kv (GQA)")
    _check(k.shape[3] == D and v.shape[3] == D and v.shape[2] == N, f"{what}: K/V shape mismatch")
    _check(D in (32, 64, 72, 80, 128, 256), f"{what}: head dim must be 32/64/72/80/128/256, got {D}")
    if out is None:
        out = torch.empty((B, H, M, D), dtype=v.dtype, device=v.device)
    else:
        _check(out.shape == (B, H, M, D) and out.dtype == v.dtype and out.device == v.device and out.is_contiguous(),
               f"{what}: out must be a contiguous [B,H,M,D] tensor of v's dtype on v's device")
    lse = torch.empty((B, H, M), dtype=torch.float32, device=v.device) if want_lse else None
    if out.numel() == 0:
        return (out, lse) if want_lse else out
    sc = (1.0 / math.sqrt(D)) if scale is None else float(scale)
    p = _lib.Fp16FwdParams(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), lse=None if lse is None else lse.data_ptr(),
        seqlens_q=None if seqlens_q is None else seqlens_q.data_ptr(),
        seqlens_k=None if seqlens_k is None else seqlens_k.data_ptr(),
        B=B, Hq=H, Hkv=Hkv, M=M, N=N, D=D, dtype=_DTYPE[q.dtype], causal=int(bool(causal)),
        window_left=int(window_left), softmax_scale=sc, backend=int(backend), **mk,
        **_gate_args(gate_flag, gate_want, q.device, what))
    with torch.cuda.device(q.device):
        ws = _status_buffer(q.device)
        rc = _lib.load().sl8_attn_fp16_fwd(C.byref(p), _ptr(ws), ws.numel() * 4, _stream(q.device))
    _lib.check(rc, "attn_fp16_fwd", 1)
    return (out, lse) if want_lse else out


def _decode_workspace(device, nbytes: int) -> torch.Tensor:
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    buf = _decode_ws.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        buf[:256].zero_()
        _decode_ws[key] = buf
    return buf


def attn_int8_decode(q, q_scale, k, k_scale, v, num_splits=-1, *, context_lens=None):
    """Reference binding csrc/fni8_api.cpp:260-263 (op csrc/kernel/attn_decode.cu:163-240)."""
    what = "superl8_b200 decode"
    if _compiled() and context_lens is None:
        r = _ext.attn_int8_decode(q, q_scale, k, k_scale, v, int(num_splits))
        _lib.launches += 2 if (r.numel() and k.shape[2] > 0) else 0
        return r
    B, H, Hkv, M, N, D = _fwd_checks(q, q_scale, k, k_scale, v, what)
    _check(v.dtype == torch.float16, f"{what}: v must be float16")
    _check(M == 1, f"{what}: query length M must be 1 (decode)")
    _check(D in (32, 64, 128, 256), f"{what}: head dim must be 32/64/128/256, got {D}")
    num_splits = int(num_splits)
    _check(num_splits != 0, f"{what}: num_splits=0 is invalid; use -1 for auto or 1..256")
    if num_splits < 0:
        num_splits = -1
    _check(num_splits <= 256, f"{what}: num_splits must be 1..256, got {num_splits}")
    if context_lens is not None:
        _check(context_lens.is_cuda and context_lens.dtype == torch.int32 and context_lens.numel() == B
               and context_lens.is_contiguous(), f"{what}: context_lens must be a contiguous int32 [B] CUDA tensor")
    out = torch.empty((B, H, 1, D), dtype=v.dtype, device=v.device)
    if out.numel() == 0:
        return out
    p = _lib.DecodeParams(
        q=q.data_ptr(), q_scale=q_scale.data_ptr(), k=k.data_ptr(), k_scale=k_scale.data_ptr(), v=v.data_ptr(),
        out=out.data_ptr(), context_lens=None if context_lens is None else context_lens.data_ptr(),
        B=B, Hq=H, Hkv=Hkv, N=N, D=D, num_splits=num_splits)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        ws = _decode_workspace(q.device, int(lib.sl8_attn_int8_decode_workspace(C.byref(p))))
        rc = lib.sl8_attn_int8_decode(C.byref(p), _ptr(ws), ws.numel(), _stream(q.device))
    _lib.check(rc, "attn_int8_decode", 2 if N > 0 else 0)
    return out


def attn_w8a8_fwd(q, q_scale, k, k_scale, v, v_scale, causal=False, causal_diag=0, per_warp_quant=True, *,
                  backend=None):
    """Full-W8A8 forward (int8 Q.K^T and int8 P.V).  Reference binding csrc/fni8_api.cpp:249-255
    (op csrc/kernel/attn_w8a8_fwd.cu:72-160): v int8 [B, Hkv, N, D], v_scale fp32 [B, Hkv, D];
    returns fp16 [B, Hq, M, D].  ``backend`` (an extension): None picks the tensor-memory kernel
    where it serves the call (D in 64/128/256, N > 0, causal diagonal at the sequence end) and the
    mma.sync kernel otherwise; SL8_BACKEND_TCGEN05 / SL8_BACKEND_MMA force one."""
    what = "superl8_b200 w8a8"
    _check(v.is_cuda and v.dtype == torch.int8, f"{what}: q/k/v must be int8")
    _check(v_scale.is_cuda and v_scale.dtype == torch.float32, f"{what}: scales must be float32")
    B, H, Hkv, M, N, D = _fwd_checks(q, q_scale, k, k_scale, v, what)
    _check(v_scale.is_contiguous() and v_scale.numel() == B * Hkv * D, f"{what}: scale shape mismatch")
    _check(D in (32, 64, 128, 256), f"{what}: head dim must be 32/64/128/256, got {D}")
    out = torch.empty((B, H, M, D), dtype=torch.float16, device=q.device)
    if out.numel() == 0:
        return out
    p = _lib.W8A8Params(q=q.data_ptr(), q_scale=q_scale.data_ptr(), k=k.data_ptr(), k_scale=k_scale.data_ptr(),
                        v=v.data_ptr(), v_scale=v_scale.data_ptr(), out=out.data_ptr(), B=B, Hq=H, Hkv=Hkv, M=M, N=N,
                        D=D, causal=int(bool(causal)), causal_diag=int(causal_diag), per_warp_quant=int(bool(per_warp_quant)))
    tc_ok = D in (64, 128, 256) and N > 0 and (not causal or int(causal_diag) == N - M)
    _check(backend in (None, _lib.SL8_BACKEND_TCGEN05, _lib.SL8_BACKEND_MMA), f"{what}: unknown backend {backend}")
    _check(tc_ok or backend != _lib.SL8_BACKEND_TCGEN05, f"{what}: the tensor-memory kernel does not serve this call")
    lib = _lib.load()
    with torch.cuda.device(q.device):
        if tc_ok and backend != _lib.SL8_BACKEND_MMA:
            ws = torch.empty(int(lib.sl8_attn_w8a8_fwd_tc_workspace(C.byref(p))), dtype=torch.uint8, device=q.device)
            rc = lib.sl8_attn_w8a8_fwd_tc(C.byref(p), _ptr(ws), ws.numel(), _stream(q.device))
        else:
            rc = lib.sl8_attn_w8a8_fwd(C.byref(p), _stream(q.device))
    _lib.check(rc, "attn_w8a8_fwd", 1)
    return out


def attn_int8_decode_kv8(q, q_scale, k, k_scale, v_i8, v_scale, num_splits=-1, *, context_lens=None):
    """Decode against an int8 K / int8 V cache.  Reference binding `attn_int8_decode_kv8`
    (kernel csrc/include/attn_decode.cuh:141-224): v_i8 int8 [B, Hkv, N, D], v_scale fp32
    [B, Hkv, D] (one scale per channel); everything else as attn_int8_decode."""
    what = "superl8_b200 decode kv8"
    _check(v_i8.is_cuda and v_i8.dtype == torch.int8, f"{what}: v must be an int8 CUDA tensor")
    _check(v_scale.is_cuda and v_scale.dtype == torch.float32, f"{what}: v_scale must be a float32 CUDA tensor")
    B, H, Hkv, M, N, D = _fwd_checks(q, q_scale, k, k_scale, v_i8, what)
    _check(M == 1, f"{what}: query length M must be 1 (decode)")
    _check(D in (32, 64, 128, 256), f"{what}: head dim must be 32/64/128/256, got {D}")
    _check(v_scale.numel() == B * Hkv * D, f"{what}: v_scale must be per-channel [B,H_kv,D]")
    num_splits = int(num_splits)
    _check(num_splits != 0, f"{what}: num_splits=0 is invalid; use -1 for auto or 1..256")
    if num_splits < 0:
        num_splits = -1
    _check(num_splits <= 256, f"{what}: num_splits must be 1..256, got {num_splits}")
    if context_lens is not None:
        _check(context_lens.is_cuda and context_lens.dtype == torch.int32 and context_lens.numel() == B
               and context_lens.is_contiguous(), f"{what}: context_lens must be a contiguous int32 [B] CUDA tensor")
    out = torch.empty((B, H, 1, D), dtype=torch.float16, device=q.device)
    if out.numel() == 0:
        return out
    v_i8, v_scale = v_i8.contiguous(), v_scale.contiguous()
    p = _lib.DecodeParams(
        q=q.data_ptr(), q_scale=q_scale.data_ptr(), k=k.data_ptr(), k_scale=k_scale.data_ptr(), v=v_i8.data_ptr(),
        out=out.data_ptr(), context_lens=None if context_lens is None else context_lens.data_ptr(),
        B=B, Hq=H, Hkv=Hkv, N=N, D=D, num_splits=num_splits)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        ws = _decode_workspace(q.device, int(lib.sl8_attn_int8_decode_workspace(C.byref(p))))
        rc = lib.sl8_attn_int8_decode_kv8(C.byref(p), v_scale.data_ptr(), _ptr(ws), ws.numel(), _stream(q.device))
    _lib.check(rc, "attn_int8_decode_kv8", 2 if N > 0 else 0)
    return out


def attn_int8_varlen(q, q_scale, k, k_scale, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, causal=False, *,
                     backend=_lib.SL8_BACKEND_AUTO):
    """Packed variable-length prefill.  Reference binding `attn_int8_varlen`
    (csrc/kernel/attn_varlen_fwd.cu:45-110): q / k int8 [total, H, D], scales fp32 [total, H],
    v fp16 [total_k, Hkv, D], cu_seqlens int32 [B + 1]; returns [total_q, Hq, D] in v's dtype."""
    what = "superl8_b200 varlen"
    for t in (q, k, v, q_scale, k_scale, cu_seqlens_q, cu_seqlens_k):
        _check(t.is_cuda, f"{what}: all inputs must be CUDA tensors")
        _check(t.device == q.device, f"{what}: all inputs must be on the same device")
    _check(q.dtype == torch.int8 and k.dtype == torch.int8, f"{what}: q/k must be int8")
    _check(q_scale.dtype == torch.float32 and k_scale.dtype == torch.float32, f"{what}: scales must be float32")
    _check(v.dtype in (torch.float16, torch.bfloat16), f"{what}: v must be float16 or bfloat16")
    _check(cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32, f"{what}: cu_seqlens must be int32")
    _check(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, f"{what}: expect [total,H,D]")
    _check(all(t.is_contiguous() for t in (q, k, v, q_scale, k_scale, cu_seqlens_q, cu_seqlens_k)),
           f"{what}: inputs must be contiguous")
    total_q, H, D = q.shape
    total_k, Hkv = k.shape[0], k.shape[1]
    B = cu_seqlens_q.numel() - 1
    _check(B >= 1 and cu_seqlens_k.numel() == B + 1, f"{what}: cu_seqlens mismatch")
    _check(Hkv > 0 and H % Hkv == 0, f"{what}: H_q must be divisible by H_kv (GQA)")
    _check(k.shape[2] == D and v.shape[2] == D and v.shape[1] == Hkv and v.shape[0] == total_k, f"{what}: K/V shape")
    _check(q_scale.numel() == total_q * H and k_scale.numel() == total_k * Hkv, f"{what}: scale shape mismatch")
    _check(D in (32, 64, 128), f"{what}: head dim must be 32/64/128, got {D}")
    out = torch.empty((total_q, H, D), dtype=v.dtype, device=v.device)
    if out.numel() == 0:
        return out
    p = _lib.VarlenParams(q=q.data_ptr(), q_scale=q_scale.data_ptr(), k=k.data_ptr(), k_scale=k_scale.data_ptr(),
                          v=v.data_ptr(), out=out.data_ptr(), cu_seqlens_q=cu_seqlens_q.data_ptr(),
                          cu_seqlens_k=cu_seqlens_k.data_ptr(), B=B, Hq=H, Hkv=Hkv, D=D, total_q=total_q,
                          total_k=total_k, max_seqlen_q=int(max_seqlen_q), v_dtype=_DTYPE[v.dtype],
                          causal=int(bool(causal)), backend=int(backend))
    with torch.cuda.device(q.device):
        ws = _status_buffer(q.device)
        rc = _lib.load().sl8_attn_int8_varlen(C.byref(p), _ptr(ws), ws.numel() * 4, _stream(q.device))
    _lib.check(rc, "attn_int8_varlen", 1)
    return out


def attn_bwd(q, k, v, o, do_, lse, scale, causal=False, *, backend=_lib.SL8_BACKEND_AUTO):
    """Reference binding csrc/fni8_api.cpp:256-259 (op csrc/kernel/attn_bwd.cu:62-109):
    (dq, dk, dv) of the attention with logits scale * q.k, from the forward's output ``o``, its
    natural-log row sums ``lse`` [B, Hq, M] and the output gradient ``do_``.  q, o, do_
    [B, Hq, M, D]; k, v [B, Hkv, N, D]; dk / dv are summed over the query heads of a KV head."""
    what = "superl8_b200 bwd"
    if _compiled() and backend == _lib.SL8_BACKEND_AUTO:
        r = _ext.attn_bwd(q, k, v, o, do_, lse, float(scale), bool(causal))
        _lib.launches += 3 if (q.numel() and k.numel()) else 0
        return r
    for t in (q, k, v, o, do_, lse):
        _check(t.is_cuda, f"{what}: all inputs must be CUDA")
        _check(t.device == q.device, f"{what}: all inputs must be on the same device")
    _check(q.dtype in (torch.float16, torch.bfloat16) and all(t.dtype == q.dtype for t in (k, v, o, do_)),
           f"{what}: q/k/v/o/do must be float16 (or all bfloat16)")
    _check(lse.dtype == torch.float32, f"{what}: lse must be float32")
    _check(all(t.dim() == 4 for t in (q, k, v, o, do_)), f"{what}: expect [B,H,S,D]")
    q, k, v, o, do_, lse = (t.contiguous() for t in (q, k, v, o, do_, lse))
    B, H, M, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    _check(Hkv > 0 and H % Hkv == 0, f"{what}: H_q must be divisible by H_kv (GQA)")
    _check(D in (32, 64, 128), f"{what}: head dim must be 32/64/128, got {D}")
    _check(k.shape == v.shape and k.shape[0] == B and k.shape[3] == D, f"{what}: K/V shape mismatch")
    _check(o.shape == q.shape and do_.shape == q.shape, f"{what}: o/do must have q's shape")
    _check(lse.numel() == B * H * M, f"{what}: lse must be [B,H,M]")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    p = _lib.BwdParams(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), dout=do_.data_ptr(),
                       lse=lse.data_ptr(), dq=dq.data_ptr(), dk=dk.data_ptr(), dv=dv.data_ptr(),
                       B=B, Hq=H, Hkv=Hkv, M=M, N=N, D=D, dtype=_DTYPE[q.dtype], causal=int(bool(causal)),
                       softmax_scale=float(scale), backend=int(backend))
    lib = _lib.load()
    with torch.cuda.device(q.device):
        nbytes = lib.sl8_attn_bwd_workspace(C.byref(p))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)   # status word; D_m = sum_d dO.O per query row
        ws[:256].zero_()
        rc = lib.sl8_attn_bwd(C.byref(p), _ptr(ws), nbytes, _stream(q.device))
        _bwd_ws[(q.device.index, torch.cuda.current_stream(q.device).cuda_stream)] = ws
    _lib.check(rc, "attn_bwd", 3 if (M and N and q.numel() and k.numel()) else 0)
    return dq, dk, dv


# ---- rotary positions and the paged int8 K/V cache (include/superl8_b200_paged.h) ----
# The compiled twin is csrc/torch_ext/sl8_torch_paged.cpp: the same checks in the same words.


def _rows(t, aligned):
    """``t`` itself when the kernels can take its rows in place, else a contiguous copy."""
    ok = (t.stride(3) == 1 or t.shape[3] == 1) and all(t.shape[d] <= 1 or t.stride(d) != 1 for d in range(3))
    if aligned and ok:
        ok = t.data_ptr() % 16 == 0 and all(t.shape[d] <= 1 or t.stride(d) % 8 == 0 for d in range(3))
    return t if ok else t.detach().clone(memory_format=torch.contiguous_format)


def _steps(t, name):
    return {f"{name}_stride_{c}": 0 if t.shape[d] == 1 else t.stride(d) for d, c in enumerate("bhs")}


def _on(t, like, what):
    _check(t.is_cuda, f"{what}: all inputs must be CUDA tensors")
    _check(t.device == like.device, f"{what}: all inputs must be on the same device")


def _rope_args(positions, inv_freq, freq_axis, like, B, S, D, what):
    """The fields that RopeParams and AppendParams share, and the rotated width."""
    _on(inv_freq, like, what)
    _check(inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous(),
           f"{what}: inv_freq must be a contiguous float32 [rot / 2] tensor")
    _check(2 * inv_freq.numel() <= D, f"{what}: 2 * len(inv_freq) must not exceed the head dim")
    f = dict(inv_freq=inv_freq.data_ptr(), rot=2 * inv_freq.numel(), n_axes=1)
    if positions is not None:
        p = positions
        shapes = f"{what}: positions must be [S], [B, S] or [axes, B, S]"
        _on(p, like, what)
        _check(p.dtype in (torch.int32, torch.int64), f"{what}: positions must be int32 or int64")
        _check(1 <= p.dim() <= 3, shapes)
        _check(p.shape[-1] == S and (p.dim() < 2 or p.shape[-2] in (B, 1)) and (p.dim() < 3 or 1 <= p.shape[0] <= 255), shapes)
        f.update(positions=p.data_ptr(), pos_is_64=int(p.dtype == torch.int64), pos_stride_s=p.stride(-1),
                 pos_stride_b=p.stride(-2) if p.dim() >= 2 and p.shape[-2] != 1 else 0,
                 pos_stride_axis=p.stride(0) if p.dim() == 3 else 0, n_axes=p.shape[0] if p.dim() == 3 else 1)
    if freq_axis is not None:
        _on(freq_axis, like, what)
        _check(freq_axis.dtype == torch.uint8 and freq_axis.dim() == 1 and freq_axis.is_contiguous()
               and freq_axis.numel() == inv_freq.numel(), f"{what}: freq_axis must be a contiguous uint8 [rot / 2] tensor")
        f.update(freq_axis=freq_axis.data_ptr())
    _check(f["n_axes"] == 1 or freq_axis is not None, f"{what}: positions with several axes need freq_axis")
    return f


def rope(q, k, positions, inv_freq, freq_axis=None, interleaved=False, inverse=False):
    """Rotary positions on q and (optionally) k [B, H, S, D]: (q_out, k_out or None).  ``inverse``
    turns by the opposite angle (the gradient)."""
    what = "superl8_b200 apply_rope"
    if _compiled():
        r = _ext.rope(q, k, positions, inv_freq, freq_axis, bool(interleaved), bool(inverse))
        _lib.launches += 1 if (r[0].numel() or (k is not None and k.numel())) else 0
        return r
    _check(q.is_cuda, f"{what}: all inputs must be CUDA tensors")
    _check(q.dim() == 4, f"{what}: expect [B,H,S,D]")
    _check(q.dtype in _DTYPE, f"{what}: q must be float16, bfloat16 or float32")
    B, Hq, S, D = q.shape
    _check(D % 2 == 0 and D > 0, f"{what}: the head dim must be even")
    q = _rows(q, False)
    q_out = torch.empty_like(q)
    f = dict(q=q.data_ptr(), q_out=q_out.data_ptr(), **_steps(q, "q"), **_steps(q_out, "q_out"), B=B, Hq=Hq, S=S, D=D)
    k_out = None
    if k is not None:
        _on(k, q, what)
        _check(k.dim() == 4 and k.shape[0] == B and k.shape[2] == S and k.shape[3] == D,
               f"{what}: q and k must agree in batch, length and head dim")
        _check(k.dtype == q.dtype, f"{what}: q and k must share one dtype")
        k = _rows(k, False)
        k_out = torch.empty_like(k)
        f.update(k=k.data_ptr(), k_out=k_out.data_ptr(), Hkv=k.shape[1], **_steps(k, "k"), **_steps(k_out, "k_out"))
    f.update(_rope_args(positions, inv_freq, freq_axis, q, B, S, D, what))
    if q.numel() or (k is not None and k.numel()):
        p = _lib.RopeParams(dtype=_DTYPE[q.dtype], interleaved=int(bool(interleaved)), inverse=int(bool(inverse)), **f)
        with torch.cuda.device(q.device):
            rc = _lib.load().sl8_rope(C.byref(p), _stream(q.device))
        _lib.check(rc, "apply_rope", 1)
    return q_out, k_out


def _paged_cache(k_i8, k_scale, v_i8, v_scale, table, lens, what):
    _check(k_i8.is_cuda, f"{what}: all inputs must be CUDA tensors")
    for t in (k_scale, v_i8, v_scale, table, lens):
        _on(t, k_i8, what)
    _check(k_i8.dtype == torch.int8 and v_i8.dtype == torch.int8, f"{what}: the cache's codes must be int8")
    _check(k_i8.dim() == 4 and k_i8.shape == v_i8.shape and k_i8.is_contiguous() and v_i8.is_contiguous(),
           f"{what}: the cache's codes must be contiguous [pages, H_kv, page_size, D], K like V")
    _check(k_scale.dtype == torch.float32 and v_scale.dtype == torch.float32, f"{what}: scales must be float32")
    _check(k_scale.dim() == 2 and k_scale.shape == k_i8.shape[:2] and k_scale.shape == v_scale.shape
           and k_scale.is_contiguous() and v_scale.is_contiguous(), f"{what}: scales must be contiguous [pages, H_kv]")
    pages, Hkv, page, D = k_i8.shape
    _check(page in (16, 32, 64, 128, 256), f"{what}: page size must be 16/32/64/128/256, got {page}")
    _check(D in (32, 64, 128, 256), f"{what}: head dim must be 32/64/128/256, got {D}")
    _check(table.dtype == torch.int32 and table.dim() == 2 and (table.shape[1] <= 1 or table.stride(1) == 1),
           f"{what}: block_table must be int32 [B, pages per sequence] with contiguous rows")
    _check(lens.dtype == torch.int32 and lens.dim() == 1 and lens.is_contiguous() and lens.shape[0] == table.shape[0],
           f"{what}: context_lens must be a contiguous int32 [B] tensor")
    return _lib.PagedCache(k=k_i8.data_ptr(), v=v_i8.data_ptr(), k_scale=k_scale.data_ptr(), v_scale=v_scale.data_ptr(),
                           block_table=table.data_ptr(), table_stride=table.stride(0), context_lens=lens.data_ptr(),
                           num_pages=pages, Hkv=Hkv, page_size=page, D=D, max_pages=table.shape[1])


def _lens_ptr(t, like, B, name, what):
    if t is None:
        return None
    _on(t, like, what)
    _check(t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous() and t.shape[0] == B,
           f"{what}: {name} must be a contiguous int32 [B] tensor")
    return t.data_ptr()


def kv_append_paged(k, v, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, new_lens=None, q=None, positions=None,
                    inv_freq=None, freq_axis=None, interleaved=False):
    """Stores new keys and values [B, H_kv, M, D] in the pages of an int8 cache (rotated on the way when
    ``inv_freq`` is given); returns the rotated q, or None without one."""
    what = "superl8_b200 kv_append_paged"
    if _compiled():
        r = _ext.kv_append_paged(k, v, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, new_lens, q, positions,
                                 inv_freq, freq_axis, bool(interleaved))
        _lib.launches += 1 if (k.numel() or (q is not None and q.numel())) else 0
        return r
    cache = _paged_cache(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, what)
    _on(k, k_i8, what)
    _on(v, k_i8, what)
    _check(k.dtype in (torch.float16, torch.bfloat16), f"{what}: k must be float16 or bfloat16")
    _check(v.dtype == k.dtype, f"{what}: k and v must share one dtype")
    _check(k.dim() == 4 and k.shape == v.shape, f"{what}: expect k and v [B,H,S,D] of one shape")
    B, Hkv, M, D = k.shape
    _check(B == context_lens.shape[0] and Hkv == cache.Hkv and D == cache.D,
           f"{what}: k and v must match the cache and block_table in batch, heads and head dim")
    f = dict(new_lens=_lens_ptr(new_lens, k_i8, B, "new_lens", what), n_axes=1)
    _check(inv_freq is not None or (q is None and positions is None and freq_axis is None),
           f"{what}: q, positions and freq_axis need inv_freq")
    if inv_freq is not None:
        f.update(_rope_args(positions, inv_freq, freq_axis, k_i8, B, M, D, what))
        _check(f["rot"] % 16 == 0, f"{what}: 2 * len(inv_freq) must be a multiple of 16")
    k, v = _rows(k, True), _rows(v, True)
    f.update(k_new=k.data_ptr(), v_new=v.data_ptr(), **_steps(k, "k"), **_steps(v, "v"))
    q_out = None
    if q is not None:
        _on(q, k_i8, what)
        _check(q.dtype == k.dtype, f"{what}: q must have the dtype of k and v")
        _check(q.dim() == 4 and q.shape[0] == B and q.shape[2] == M and q.shape[3] == D,
               f"{what}: q must be [B,H_q,S,D] with the batch, length and head dim of k")
        q = _rows(q, True)
        q_out = torch.empty_like(q)
        f.update(q=q.data_ptr(), q_out=q_out.data_ptr(), Hq=q.shape[1], **_steps(q, "q"), **_steps(q_out, "q_out"))
    if k.numel() or (q is not None and q.numel()):
        p = _lib.AppendParams(B=B, M=M, dtype=_DTYPE[k.dtype], interleaved=int(bool(interleaved)), **f)
        with torch.cuda.device(k_i8.device):
            rc = _lib.load().sl8_kv_append_paged(C.byref(cache), C.byref(p), _stream(k_i8.device))
        _lib.check(rc, "kv_append_paged", 1)
    return q_out


def kv_read_paged(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, num_tokens, first=None, dtype=torch.float16):
    """Tokens first[b] ... first[b] + num_tokens - 1 of every sequence as 16-bit (k, v) [B, H_kv, num_tokens, D]."""
    what = "superl8_b200 kv_read_paged"
    _check(dtype in (torch.float16, torch.bfloat16), f"{what}: dtype must be float16 or bfloat16")
    if _compiled():
        r = _ext.kv_read_paged(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, int(num_tokens), first,
                               dtype == torch.bfloat16)
        _lib.launches += 1 if r[0].numel() else 0
        return r
    cache = _paged_cache(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, what)
    _check(0 <= int(num_tokens) <= 0x7fffffff, f"{what}: num_tokens must not be negative")
    B = context_lens.shape[0]
    start = _lens_ptr(first, k_i8, B, "first", what)
    k = torch.empty((B, cache.Hkv, int(num_tokens), cache.D), dtype=dtype, device=k_i8.device)
    v = torch.empty_like(k)
    if k.numel():
        with torch.cuda.device(k_i8.device):
            rc = _lib.load().sl8_kv_read_paged(C.byref(cache), B, start, int(num_tokens), _DTYPE[dtype], k.data_ptr(),
                                               v.data_ptr(), _stream(k_i8.device))
        _lib.check(rc, "kv_read_paged", 1)
    return k, v


def attn_paged(q, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, scale=None, causal=True, window_left=-1,
               query_lens=None, max_context_len=0, backend=_lib.SL8_BACKEND_AUTO):
    """Attention of q [B, H_q, M, D] over a paged int8 cache; output like q."""
    what = "superl8_b200 attn_paged_cached"
    window_left = -1 if window_left < 0 else min(int(window_left), 0x7fffffff)
    limit = 0 if max_context_len is None else max(0, min(int(max_context_len), 0x7fffffff))
    if _compiled():
        r = _ext.attn_paged(q, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, None if scale is None else float(scale),
                            bool(causal), window_left, query_lens, limit, int(backend))
        _lib.launches += 2 if r.numel() else 0
        return r
    cache = _paged_cache(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, what)
    _on(q, k_i8, what)
    _check(q.dtype in (torch.float16, torch.bfloat16), f"{what}: q must be float16 or bfloat16")
    _check(q.dim() == 4, f"{what}: expect q [B,H,S,D]")
    B, Hq, M, D = q.shape
    _check(B == context_lens.shape[0] and D == cache.D, f"{what}: q must match the cache and block_table in batch and head dim")
    _check(cache.Hkv > 0 and Hq % cache.Hkv == 0, f"{what}: H_q must be divisible by H_kv (GQA)")
    qlens = _lens_ptr(query_lens, k_i8, B, "query_lens", what)
    q = _rows(q, True)
    out = torch.empty_like(q)
    if out.numel() == 0:
        return out
    p = _lib.PagedAttnParams(q=q.data_ptr(), out=out.data_ptr(), **_steps(q, "q"), **_steps(out, "out"), query_lens=qlens, B=B,
                             Hq=Hq, M=M, dtype=_DTYPE[q.dtype], causal=int(bool(causal)), window_left=window_left,
                             max_context_len=limit, softmax_scale=(1.0 / math.sqrt(D)) if scale is None else float(scale), backend=int(backend))
    lib = _lib.load()
    with torch.cuda.device(q.device):
        nbytes = int(lib.sl8_attn_paged_workspace(C.byref(cache), C.byref(p)))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        rc = lib.sl8_attn_paged(C.byref(cache), C.byref(p), _ptr(ws), nbytes, _stream(q.device))
    _lib.check(rc, "attn_paged_cached", 2)
    return out
