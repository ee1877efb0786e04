"""Autograd wrapper of the fused cross attention (``csrc/cross_attention_*.cu``) and of the decoding-step attention over a shared
prompt (``csrc/step_attention.cu``)."""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad

from . import native as N
from .native_sequence_loss import address, bind, current_stream, first_derivative, on_device

_SIGNATURES = {                      # p: pointer; the stream is the last one
    "sb_cross_attention_fwd": "pppppp",
    "sb_cross_attention_bwd": "pppppppppp",
    "sb_cross_attention_workspace": "p",
    "sb_shared_prefix_workspace": "pp",
    "sb_shared_prefix_attention": "ppppp",
}


# The C structures' fields, packed (filling a ctypes structure takes 1.3 us instead of 0.3).
# SbCrossAttention: q, k, v; strides (batch, time, head) of each; lengths, mask; type, M, G, rep, Tq, Tk, Hk, D; scale
_ATTENTION = struct.Struct("=3Q9q2Q8if4x")
# SbOwnCache: k, v; strides (batch, time, head) of each; lengths; size
_OWN = struct.Struct("=2Q6qQi4x")


def _call(name):
    f = bind(name, _SIGNATURES)
    if name.endswith("_workspace"):
        f.restype = ctypes.c_longlong
    return f


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself if the kernels can address it (contiguous head rows on 16-byte boundaries), else a dense copy of its own."""
    sb, st, sh, sd = t.stride()
    if sd == 1 and not (sb | st | sh) & 7 and not t.data_ptr() & 15:
        nb, nt, nh, _ = t.shape
        if (sb > 0 or nb == 1) and (st > 0 or nt == 1) and (sh > 0 or nh == 1):
            return t
    # not contiguous(): that is the same tensor for a dense view at an odd offset, or with odd strides of axes of size one
    return t.clone(memory_format=torch.contiguous_format)


def _lengths(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None or (t.dtype == torch.int32 and t.is_contiguous()):
        return t
    # clamped in 64 bits before the narrowing, so that a 64-bit length cannot wrap and a type without the bound need not hold it
    return t.long().clamp(0, 2 ** 31 - 1).to(torch.int32).contiguous()


def _block(q, k, v, lengths, mask, scale) -> bytes:
    B, Tq, H, D = q.shape
    M, Tk, Hk, _ = k.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    return _ATTENTION.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                           address(lengths), address(mask), 0 if q.dtype == torch.bfloat16 else 1, M, B // M, H // Hk, Tq, Tk, Hk, D, scale)


def _scratch(nbytes: int, what: str, device) -> Optional[torch.Tensor]:
    if nbytes < 0:
        raise RuntimeError(f"speech_b200 native call {what} refused its arguments")
    return torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None


def _forward(q, k, v, lengths, mask, scale, for_backward):
    """The output and, for a backward pass, one buffer: what rounding took from the output (16 bits), then lse."""
    B, Tq, H, D = q.shape
    p = _block(q, k, v, lengths, mask, scale)
    out = q.new_empty((B, Tq, H * D))
    kept, rest, lse = None, 0, 0
    if for_backward:
        rows = B * Tq * H
        kept = q.new_empty(rows * (D // 2 + 1), dtype=torch.float32)
        rest = kept.data_ptr()
        lse = rest + rows * D * 2
    ws = _scratch(_call("sb_cross_attention_workspace")(p), "sb_cross_attention_workspace", q.device)
    N._check(_call("sb_cross_attention_fwd")(p, out.data_ptr(), rest, lse, address(ws), current_stream()), "sb_cross_attention_fwd")
    return out, kept


def _backward(ctx, dout):
    q, k, v, out, lengths, mask, kept = ctx.saved_tensors
    if not dout.is_contiguous() or dout.data_ptr() & 15:
        dout = dout.clone(memory_format=torch.contiguous_format)
    want_q, want_k, want_v = ctx.needs_input_grad[:3]
    B, Tq, H, D = q.shape
    with on_device(q):
        M, Hk = k.shape[0], k.shape[2]
        units = M * Hk
        # statistics in lines of a multiple of 64, a maximum per 128 rows that read the same keys, in fp16 one per 64 keys
        norms = (k.shape[1] + 63) // 64 if q.dtype == torch.float16 else 0
        ws = q.new_empty(2 * B * H * ((Tq + 63) // 64 * 64) + units * ((B * H * Tq // units + 127) // 128 + norms), dtype=torch.float32)
        dq = q.new_empty(q.shape) if want_q else None
        dk = k.new_empty(k.shape) if want_k or want_v else None
        dv = v.new_empty(v.shape) if want_k or want_v else None
        g = _block(q, k, v, lengths, mask, ctx.scale)
        rest = kept.data_ptr()
        N._check(_call("sb_cross_attention_bwd")(g, out.data_ptr(), rest, dout.data_ptr(), rest + B * Tq * H * D * 2, ws.data_ptr(),
                                                 address(dq), address(dk), address(dv), current_stream()), "sb_cross_attention_bwd")
    return dq, dk if want_k else None, dv if want_v else None, None, None, None


def _has_tangent(*tensors) -> bool:
    """Whether forward-mode differentiation is on for one of them; such a tensor need not require a gradient."""
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _CrossAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale):
        out, kept = _forward(q, k, v, lengths, mask, scale, True)
        ctx.save_for_backward(q, k, v, out, lengths, mask, kept)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        return first_derivative(_backward, ctx, dout)


def cross_attention(q, k, v, key_lengths=None, key_mask=None, scale=None):
    D, Tk = q.shape[3], k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if D % 8 or D > 128 or Tk == 0 or q.numel() == 0 or not 0.0 < scale < 1e30 or _has_tangent(q, k, v):
        from . import reference

        return reference.cross_attention(q, k, v, key_lengths, key_mask, scale)
    with on_device(q):
        q, k, v = _rows(q), _rows(k), _rows(v)
        lengths, mask = _lengths(key_lengths), None if key_mask is None else key_mask.contiguous()
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return _CrossAttentionFn.apply(q, k, v, lengths, mask, scale)
        return _forward(q, k, v, lengths, mask, scale, False)[0]


def shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, prefix_lengths=None, scale=None):
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_prefix, v_prefix, k, v)):
        raise RuntimeError("shared_prefix_attention has no backward pass on GPUs: call it under torch.no_grad() or on detached tensors")
    if _has_tangent(q, k_prefix, v_prefix, k, v):
        raise RuntimeError("shared_prefix_attention has no forward-mode derivative on GPUs")
    B, Tq, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if D % 8 or D > 128 or q.numel() == 0 or k_prefix.shape[1] == 0 or k.shape[1] == 0 or not 0.0 < scale < 1e30:
        from . import reference

        return reference.shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, prefix_lengths, scale)
    with on_device(q):
        q, kp, vp, k, v = _rows(q), _rows(k_prefix), _rows(v_prefix), _rows(k), _rows(v)
        lengths, prefix_lengths = _lengths(lengths), _lengths(prefix_lengths)
        p = _block(q, kp, vp, prefix_lengths, None, scale)
        ks, vs = k.stride(), v.stride()
        o = _OWN.pack(k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], lengths.data_ptr(), k.shape[1])
        out = q.new_empty((B, Tq, H * D))
        ws = _scratch(_call("sb_shared_prefix_workspace")(p, o), "sb_shared_prefix_workspace", q.device)
        N._check(_call("sb_shared_prefix_attention")(p, o, out.data_ptr(), address(ws), current_stream()), "sb_shared_prefix_attention")
        return out
