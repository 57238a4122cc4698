"""Autograd wrapper with the reference's shape (reference superl8/autograd.py:48-108):
forward = quantised int8 kernel (saving out and the natural-log LSE), backward =
the exact FlashAttention-2 gradient, straight-through w.r.t. the quantisation;
``attn_ref`` = the reference's gradcheck twin (plain forward, the same analytic backward)."""

from __future__ import annotations

import math

import torch

from . import _C, _lib
from .quant import quantize_qk


def _softmax_scale(d: int, scale):
    return (1.0 / math.sqrt(d)) if scale is None else scale


def _attn_backward(q, k, v, out, d_out, causal, scale):
    """Exact FlashAttention-2 gradient in fp32 torch ops (reference superl8/autograd.py:29-45);
    all tensors [B, H, S, D] with equal head counts.  Serves ``attn_ref`` only (gradcheck in
    fp64/fp32 on whatever device the tensors live on); ``attn`` uses the CUDA kernels."""
    qf, kf, vf, of, dof = (t.float() if t.dtype in (torch.float16, torch.bfloat16) else t for t in (q, k, v, out, d_out))
    s = torch.einsum("bhmd,bhnd->bhmn", qf, kf) * scale
    if causal:
        m, n = s.shape[-2], s.shape[-1]
        keep = torch.ones(m, n, device=s.device, dtype=torch.bool).tril(n - m)
        s = s.masked_fill(~keep, float("-inf"))
    p = torch.softmax(s, dim=-1)
    dv = torch.einsum("bhmn,bhmd->bhnd", p, dof)
    dp = torch.einsum("bhmd,bhnd->bhmn", dof, vf)
    drow = (dof * of).sum(dim=-1, keepdim=True)
    ds = p * (dp - drow)
    dq = torch.einsum("bhmn,bhnd->bhmd", ds, kf) * scale
    dk = torch.einsum("bhmn,bhmd->bhnd", ds, qf) * scale
    return dq, dk, dv


class _AttnInt8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, scale):
        scale = _softmax_scale(q.shape[-1], scale)
        q_i8, q_scale, k_i8, k_scale, k_mean = quantize_qk(q, k, softmax_scale=scale)
        out, lse = _C.attn_int8_fwd_train(q_i8, q_scale.squeeze(-1).contiguous(), k_i8,
                                          k_scale.squeeze(-1).contiguous(), v.contiguous(), causal)
        # The kernel saw the SMOOTHED keys, so its row statistic is log sum exp(scale q.(k - mean)):
        # the true one minus scale * q.mean.  The backward recomputes the logits from the
        # unsmoothed k, so the saved statistic gets that term back (the reference saves the
        # kernel's value as it is, superl8/autograd.py:56-66, and its gradients are off by
        # exp(scale q.mean) per row whenever K carries a per-channel mean).
        g = q.shape[1] // k.shape[1]
        km = k_mean.squeeze(-2).repeat_interleave(g, dim=1) if g > 1 else k_mean.squeeze(-2)   # [B, Hq, D]
        lse = lse + scale * torch.einsum("bhmd,bhd->bhm", q.float(), km)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    def backward(ctx, d_out):
        q, k, v, out, lse = ctx.saved_tensors
        from .ops import backward_cuda

        dq, dk, dv = backward_cuda(q, k, v, out, lse, d_out, causal=ctx.causal, scale=ctx.scale)
        return dq, dk, dv, None, None


class _AttnRef(torch.autograd.Function):
    """Plain (non-quantised) forward with the same analytic backward: the gradient mathematics
    can be checked with torch.autograd.gradcheck (reference superl8/autograd.py:77-98)."""

    @staticmethod
    def forward(ctx, q, k, v, causal, scale):
        scale = _softmax_scale(q.shape[-1], scale)
        s = torch.einsum("bhmd,bhnd->bhmn", q, k) * scale
        if causal:
            m, n = s.shape[-2], s.shape[-1]
            keep = torch.ones(m, n, device=s.device, dtype=torch.bool).tril(n - m)
            s = s.masked_fill(~keep, float("-inf"))
        out = torch.einsum("bhmn,bhnd->bhmd", torch.softmax(s, dim=-1), v)
        ctx.save_for_backward(q, k, v, out)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    def backward(ctx, d_out):
        q, k, v, out = ctx.saved_tensors
        dq, dk, dv = _attn_backward(q, k, v, out, d_out, ctx.causal, ctx.scale)
        return dq.to(q.dtype), dk.to(k.dtype), dv.to(v.dtype), None, None


def attn(q, k, v, *, causal: bool = False, scale: float | None = None):
    """Differentiable int8 attention (reference superl8/autograd.py:101-103)."""
    return _AttnInt8.apply(q, k, v, causal, scale)


def attn_ref(q, k, v, *, causal: bool = False, scale: float | None = None):
    """Non-quantised attention sharing the analytic backward (reference superl8/autograd.py:106-108)."""
    return _AttnRef.apply(q, k, v, causal, scale)


class _Rope(torch.autograd.Function):
    """apply_rope's gradient under the ctypes binding (the compiled one has its own): the rotation is linear and
    orthogonal, so its gradient is the rotation by the opposite angle, itself differentiable the same way."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, freq_axis, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq, freq_axis)
        ctx.interleaved, ctx.inverse = interleaved, inverse
        return _C.rope(q, k, positions, inv_freq, freq_axis, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq, freq_axis = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[:2]
        dq, dk = (dq if need_q else None), (dk if need_k else None)
        if dq is None and dk is None:
            return (None,) * 7
        args = (positions, inv_freq, freq_axis, ctx.interleaved, not ctx.inverse)
        first, second = (dq, dk) if dq is not None else (dk, None)
        a, b = _Rope.apply(first, second, *args)
        return (a, b, None, None, None, None, None) if dq is not None else (None, a, None, None, None, None, None)


def apply_rope(q, k, positions, inv_freq, *, freq_axis=None, interleaved: bool = False):
    """Rotary positions on q [B, Hq, S, D] and k [B, Hkv, S, D] (``k`` may be None): (q_out, k_out).

    Channel pair i of a row turns by ``positions[axis(i)] * inv_freq[i]``: pairs are channels
    (i, i + rot/2) with rot = 2 len(inv_freq), or (2i, 2i + 1) with ``interleaved``; channels from rot on
    stay.  ``positions``: int32 / int64 [S], [B, S], or [axes, B, S] with ``freq_axis`` (uint8 [rot/2])
    naming the axis of every frequency -- time, height and width for images and video (see
    :func:`rope_freq_axis`).  fp16 / bf16 / fp32, any even D, strided views with contiguous channels in
    place.  Angles are formed in 64 bits, so far positions keep their precision.  Differentiable in q and
    k (also twice); ``inv_freq`` is a constant.  What it returns is what ``attn``, ``attn_int8_fwd`` and the
    other prefill operators take; ``kv_append_paged`` does the same rotation on the way into a cache."""
    if _C._compiled():
        r = _C._ext.apply_rope(q, k, positions, inv_freq, freq_axis, bool(interleaved))
        _lib.launches += 1 if (r[0].numel() or (k is not None and k.numel())) else 0
        return r
    if inv_freq.requires_grad:
        raise RuntimeError("superl8_b200 apply_rope: inv_freq is a constant (no gradient is computed for it)")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rope.apply(q, k, positions, inv_freq, freq_axis, bool(interleaved), False)
    return _C.rope(q, k, positions, inv_freq, freq_axis, interleaved)


def rope_freq_axis(sections, *, mixed: bool = False, device=None) -> torch.Tensor:
    """uint8 [sum(sections)]: the axis of every frequency when axis a owns ``sections[a]`` of them -- in
    blocks (all of axis 0, then axis 1, ...), or ``mixed``: dealt out in turn (0, 1, 2, 0, 1, 2, ...)
    until an axis has its share."""
    sections = [int(n) for n in sections]
    if not sections or len(sections) > 255 or min(sections) < 0:
        raise ValueError("superl8_b200 rope_freq_axis: sections must be 1 to 255 numbers >= 0")
    if mixed:
        order = sorted((i, a) for a, n in enumerate(sections) for i in range(n))
        axis = [a for _, a in order]
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(axis, dtype=torch.uint8, device=device)
