"""Autograd wrappers of the policy and preference losses (``csrc/sequence_loss.cu``)."""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import native as N

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_KINDS = {"dpo": 0, "ipo": 1, "rpo_sq": 2}
_SIGNATURES = {                      # p: pointer, l: 64-bit integer, i: integer, f: float; the stream is the last pointer
    "sb_policy_loss_fwd": "pilllppppp" + "liii" + "fff" + "ppppppp" + "p",
    "sb_preference_loss_fwd": "pilllppp" + "liii" + "if" + "ppppppp" + "p",
    "sb_sequence_loss_bwd": "pilllpp" + "liii" + "pppp" + "ip" + "p",
}
_C = {"p": ctypes.c_void_p, "l": ctypes.c_longlong, "i": ctypes.c_int, "f": ctypes.c_float}
_bound: dict = {}


def bind(name: str, signatures=None):
    """The library's entry point with its argument types declared once: plain Python numbers are then converted by ctypes itself,
    a few microseconds less per call than wrapping each of twenty-odd arguments."""
    f = _bound.get(name)
    if f is None:
        f = getattr(N.lib(), name)
        f.argtypes = [_C[c] for c in (signatures or _SIGNATURES)[name]]
        _bound[name] = f
    return f


def current_stream() -> int:
    return N._stream().value or 0


def on_device(t: torch.Tensor):
    """Makes the tensor's device current for the launches of the block (nothing to do in the usual case)."""
    index = t.device.index
    current = N._cur_device() if N._cur_device is not None else torch.cuda.current_device()
    return contextlib.nullcontext() if index == current else torch.cuda.device(index)


def first_derivative(f, ctx, *grads):
    """Runs a backward pass that cannot be differentiated itself: under ``create_graph`` its results raise when that is tried."""
    if torch.is_grad_enabled():
        return once_differentiable(f)(ctx, *grads)
    return f(ctx, *grads)


def address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _layout(logits: torch.Tensor):
    """(type code, element strides of n, t, c) and (N, T, C, V) of logits whose last axis is contiguous."""
    if logits.dim() == 3:
        (n, t, v), (sn, st, _) = logits.shape, logits.stride()
        return (_TYPES[logits.dtype], sn, st, 0), (n, t, 1, v)
    sn, st, sc, _ = logits.stride()
    return (_TYPES[logits.dtype], sn, st, sc), tuple(logits.shape)


def _plain(t: Optional[torch.Tensor], dtype: torch.dtype) -> Optional[torch.Tensor]:
    """A tensor that takes no gradient, dense and of the kernels' type."""
    if t is None:
        return None
    if t.requires_grad:
        t = t.detach()
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _mask8(mask: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    return _plain(mask if mask.dtype == torch.bool else mask != 0, torch.bool)      # one byte per position


_max_blocks = 0


def _blocks() -> int:
    global _max_blocks
    if not _max_blocks:
        _max_blocks = int(N.lib().sb_sequence_loss_blocks())
    return _max_blocks


def _gradient(upstream, logits, targets, mask, lse, slope, seq_slope, out, unless_one):
    """``lse``, ``slope``, ``seq_slope``: addresses."""
    layout, sizes = _layout(logits)
    g = _plain(upstream, torch.float32)
    with on_device(logits):
        N._check(bind("sb_sequence_loss_bwd")(logits.data_ptr(), *layout, targets.data_ptr(), address(mask), *sizes, lse, slope, seq_slope, g.data_ptr(),
                                              unless_one, out.data_ptr(), current_stream()), "sb_sequence_loss_bwd")
    return out


def _policy_backward(ctx, dloss, _):
    logits, targets, mask, kept, grad = ctx.saved_tensors
    first, ctx.first = ctx.first, False
    # handed out with a version counter of its own: what its owner does to it is nothing to a further backward pass, which does not read it
    out = grad.data if first else logits.new_empty(logits.shape)
    lse = kept.data_ptr() + 8 * _blocks() + 8
    return _gradient(dloss, logits, targets, mask, lse, lse + 8 * targets.numel(), 0, out, int(first)), None, None, None, None, None, None, None, None, None


class _PolicyLossFn(torch.autograd.Function):
    """The forward kernel writes the gradient for an upstream gradient of 1 while it has the row; the first backward pass hands that
    buffer out (rewritten on the device if the upstream gradient is another one), a further one computes a new buffer."""

    @staticmethod
    def forward(ctx, logits, targets, mask, old, adv, ref, lo, hi, kl_beta, want_grad):
        rows = targets.numel()
        loss = logits.new_empty((), dtype=torch.float32)
        logp = logits.new_empty(targets.shape, dtype=torch.float32)
        kept = logits.new_empty(2 * _blocks() + 2 + 3 * rows, dtype=torch.float32)       # fp64 sums of the blocks and the count, lse (two parts), slopes
        ws = kept.data_ptr()
        lse = ws + 8 * _blocks() + 8
        grad = logits.new_empty(logits.shape) if want_grad else None
        layout, sizes = _layout(logits)
        N._check(bind("sb_policy_loss_fwd")(logits.data_ptr(), *layout, targets.data_ptr(), address(mask), old.data_ptr(), address(ref), adv.data_ptr(), *sizes,
                                            lo, hi, kl_beta, ws + 8 * _blocks(), ws, loss.data_ptr(), logp.data_ptr(), lse, lse + 8 * rows, address(grad),
                                            current_stream()), "sb_policy_loss_fwd")
        if want_grad:
            ctx.save_for_backward(logits, targets, mask, kept, grad)
            ctx.first = True
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    def backward(ctx, dloss, dlogp):
        return first_derivative(_policy_backward, ctx, dloss, dlogp)


def _preference_backward(ctx, dloss, _):
    logits, targets, mask, kept = ctx.saved_tensors
    rows = targets.numel()
    lse = kept.data_ptr() + 8 * (rows + logits.shape[0])
    out = logits.new_empty(logits.shape)
    return _gradient(dloss, logits, targets, mask, lse, 0, lse + 8 * rows, out, 0), None, None, None, None, None, None


class _PreferenceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, ref, beta, kind, gap):
        rows, n = targets.numel(), logits.shape[0]
        loss = logits.new_empty((), dtype=torch.float32)
        rewards = logits.new_empty(n, dtype=torch.float32)
        # log ratios of the positions and of the sequences (fp64), lse (two parts) and the slopes of the sequences (fp32)
        kept = logits.new_empty(4 * rows + 3 * n, dtype=torch.float32)
        ws = kept.data_ptr()
        lse = ws + 8 * (rows + n)
        layout, sizes = _layout(logits)
        N._check(bind("sb_preference_loss_fwd")(logits.data_ptr(), *layout, targets.data_ptr(), address(mask), ref.data_ptr(), *sizes, kind, beta, address(gap),
                                                ws, ws + 8 * rows, loss.data_ptr(), rewards.data_ptr(), lse + 8 * rows, lse, current_stream()),
                 "sb_preference_loss_fwd")
        ctx.save_for_backward(logits, targets, mask, kept)
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    def backward(ctx, dloss, drewards):
        return first_derivative(_preference_backward, ctx, dloss, drewards)


def policy_loss(logits, targets, mask, old_logp, advantages, ref_logp=None, clip=0.2, clip_high=None, kl_beta=0.0):
    with on_device(logits):
        x = logits if logits.stride(-1) == 1 else logits.contiguous()
        want = torch.is_grad_enabled() and logits.requires_grad
        f32 = torch.float32
        return _PolicyLossFn.apply(x, _plain(targets, torch.int64), _mask8(mask), _plain(old_logp, f32), _plain(advantages, f32), _plain(ref_logp, f32),
                                   float(clip), float(clip if clip_high is None else clip_high), float(kl_beta), want)


def preference_loss(logits, targets, mask, ref_logp, beta=0.1, loss_type="dpo", reward_gap=None):
    with on_device(logits):
        x = logits if logits.stride(-1) == 1 else logits.contiguous()
        return _PreferenceLossFn.apply(x, _plain(targets, torch.int64), _mask8(mask), _plain(ref_logp, torch.float32), float(beta), _KINDS[loss_type],
                                       _plain(reward_gap, torch.float32))
