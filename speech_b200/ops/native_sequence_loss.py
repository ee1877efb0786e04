"""Autograd wrappers of the policy and preference losses (``csrc/sequence_loss.cu``)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .native import _check, _ptr, _stream, lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_KINDS = {"dpo": 0, "ipo": 1, "rpo_sq": 2}


_max_blocks = 0


def _blocks() -> int:
    global _max_blocks
    if not _max_blocks:
        _max_blocks = int(lib().sb_sequence_loss_blocks())
    return _max_blocks


def _layout(logits: torch.Tensor):
    """Type code, element strides of (n, t, c) and sizes of logits whose last axis is contiguous."""
    if logits.dim() == 3:
        (n, t, v), (sn, st, _), c, sc = logits.shape, logits.stride(), 1, 0
    else:
        (n, t, c, v), (sn, st, sc, _) = logits.shape, logits.stride()
    ll, i = ctypes.c_longlong, ctypes.c_int
    return (i(_TYPES[logits.dtype]), ll(sn), ll(st), ll(sc)), (ll(n), i(t), i(c), i(v))


def _f32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.detach().to(torch.float32).contiguous()


def _mask8(mask: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    return (mask if mask.dtype == torch.bool else mask != 0).contiguous()      # one byte per position


def _gradient(ctx, upstream, logits, targets, mask, lse, slope, seq_slope, out, unless_one):
    layout, sizes = _layout(logits)
    g = upstream.detach().to(torch.float32).contiguous()
    _check(lib().sb_sequence_loss_bwd(_ptr(logits), *layout, _ptr(targets), _ptr(mask), *sizes, _ptr(lse), _ptr(slope), _ptr(seq_slope), _ptr(g),
                                      ctypes.c_int(unless_one), _ptr(out), _stream()), "sb_sequence_loss_bwd")
    return out


class _PolicyLossFn(torch.autograd.Function):
    """The forward kernel writes the gradient for an upstream gradient of 1 while it has the row; the first backward pass hands that
    buffer out (rewritten on the device if the upstream gradient is another one), a further one computes a new buffer."""

    @staticmethod
    def forward(ctx, logits, targets, mask, old, adv, ref, lo, hi, kl_beta, want_grad):
        dev, rows = logits.device, targets.numel()
        f32 = dict(dtype=torch.float32, device=dev)
        loss, logp, stats = torch.empty((), **f32), torch.empty(targets.shape, **f32), torch.empty((2, rows), **f32)
        lse, slope = stats.unbind(0)
        ws = torch.empty(_blocks() + 1, dtype=torch.float64, device=dev)          # sums of the blocks, and the count
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
        layout, sizes = _layout(logits)
        _check(lib().sb_policy_loss_fwd(_ptr(logits), *layout, _ptr(targets), _ptr(mask), _ptr(old), _ptr(ref), _ptr(adv), *sizes, ctypes.c_float(lo),
                                        ctypes.c_float(hi), ctypes.c_float(kl_beta), ctypes.c_void_p(ws.data_ptr() + 8 * _blocks()), _ptr(ws), _ptr(loss), _ptr(logp), _ptr(lse),
                                        _ptr(slope), _ptr(grad), _stream()), "sb_policy_loss_fwd")
        if want_grad:
            ctx.save_for_backward(logits, targets, mask, lse, slope)
            ctx.grad = grad
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        logits, targets, mask, lse, slope = ctx.saved_tensors
        out, ctx.grad = ctx.grad, None
        first = out is not None
        if not first:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return (_gradient(ctx, dloss, logits, targets, mask, lse, slope, None, out, int(first)),) + (None,) * 9


class _PreferenceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, ref, beta, kind, gap):
        dev, rows, n = logits.device, targets.numel(), logits.shape[0]
        f32 = dict(dtype=torch.float32, device=dev)
        loss, rewards, seq_slope, lse = torch.empty((), **f32), torch.empty(n, **f32), torch.empty(n, **f32), torch.empty(rows, **f32)
        ws = torch.empty(rows + n, dtype=torch.float64, device=dev)               # log ratios of the positions and of the sequences
        layout, sizes = _layout(logits)
        _check(lib().sb_preference_loss_fwd(_ptr(logits), *layout, _ptr(targets), _ptr(mask), _ptr(ref), *sizes, ctypes.c_int(kind), ctypes.c_float(beta),
                                            _ptr(gap), _ptr(ws), ctypes.c_void_p(ws.data_ptr() + 8 * rows), _ptr(loss), _ptr(rewards), _ptr(seq_slope), _ptr(lse),
                                            _stream()), "sb_preference_loss_fwd")
        ctx.save_for_backward(logits, targets, mask, lse, seq_slope)
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        logits, targets, mask, lse, seq_slope = ctx.saved_tensors
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return (_gradient(ctx, dloss, logits, targets, mask, lse, None, seq_slope, out, 0),) + (None,) * 6


def policy_loss(logits, targets, mask, old_logp, advantages, ref_logp=None, clip=0.2, clip_high=None, kl_beta=0.0):
    with torch.cuda.device(logits.device):
        x = logits if logits.stride(-1) == 1 else logits.contiguous()
        want = torch.is_grad_enabled() and logits.requires_grad
        return _PolicyLossFn.apply(x, targets.to(torch.int64).contiguous(), _mask8(mask), _f32(old_logp), _f32(advantages), _f32(ref_logp), float(clip),
                                   float(clip if clip_high is None else clip_high), float(kl_beta), want)


def preference_loss(logits, targets, mask, ref_logp, beta=0.1, loss_type="dpo", reward_gap=None):
    with torch.cuda.device(logits.device):
        x = logits if logits.stride(-1) == 1 else logits.contiguous()
        return _PreferenceLossFn.apply(x, targets.to(torch.int64).contiguous(), _mask8(mask), _f32(ref_logp), float(beta), _KINDS[loss_type], _f32(reward_gap))
