"""Hot-op entry points used by the model code.

Every function here has two implementations: the hand-written sm_100a kernels in
``speech_b200/ops/csrc`` (bound through ``speech_b200.ops.native``), used for CUDA tensors, and
the plain-PyTorch statement in ``speech_b200.ops.reference``, used on the CPU and as the test
oracle.  On a machine with a GPU the kernels are mandatory: if the extension library is missing,
the first CUDA call raises instead of silently falling back to library kernels
(set ``SPEECH_B200_ALLOW_EAGER=1`` to run the eager reference math on a GPU on purpose, which is
what the ``--impl eager`` arm of the benchmark does).
"""
from __future__ import annotations

import contextlib
import os
import threading
from typing import Optional

import torch

from . import reference

_state = threading.local()


def get_compute_dtype() -> Optional[torch.dtype]:
    return getattr(_state, "dtype", None)


@contextlib.contextmanager
def compute_dtype(dtype: Optional[torch.dtype]):
    """Activations inside the block run in ``dtype`` (bf16 on GPUs); master weights stay fp32."""
    prev = getattr(_state, "dtype", None)
    _state.dtype = dtype
    try:
        yield
    finally:
        _state.dtype = prev


_env_eager = [os.environ.get("SPEECH_B200_ALLOW_EAGER", "0") == "1", 0]


def eager_allowed() -> bool:
    # the environment is re-read only every 4096 calls: this predicate runs once per op
    _env_eager[1] += 1
    if _env_eager[1] & 4095 == 1:
        _env_eager[0] = os.environ.get("SPEECH_B200_ALLOW_EAGER", "0") == "1"
    return _env_eager[0] or getattr(_state, "eager", False)


@contextlib.contextmanager
def eager_mode(enabled: bool = True):
    """Force the plain-PyTorch math even for CUDA tensors (baseline arm / debugging)."""
    prev = getattr(_state, "eager", False)
    _state.eager = enabled
    try:
        yield
    finally:
        _state.eager = prev


_native = None
_native_err: Optional[BaseException] = None


def _nat():
    """The ctypes binding module, loaded on first use."""
    global _native, _native_err
    if _native is None and _native_err is None:
        try:
            from . import native as _n  # noqa: F811

            _n.load()
            _native = _n
        except BaseException as e:  # noqa: BLE001
            _native_err = e
    if _native is None:
        raise RuntimeError(
            "speech_b200 native kernels are not available "
            f"({_native_err!r}). Build them with `python -m speech_b200.ops.build` "
            "or set SPEECH_B200_ALLOW_EAGER=1 to run the eager reference math."
        )
    return _native


def native_available() -> bool:
    try:
        _nat()
        return True
    except RuntimeError:
        return False


def _use_native(t: torch.Tensor) -> bool:
    if not t.is_cuda or eager_allowed():
        return False
    _nat()  # raises loudly when the library is missing on a GPU machine
    return True


def lowp(param: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Working copy of a master weight in the compute dtype (the optimizer arena keeps one up to date)."""
    dtype = dtype or get_compute_dtype()
    if dtype is None or param.dtype == dtype:
        return param
    lp = getattr(param, "_lowp", None)
    if lp is not None and lp.dtype == dtype and lp.device == param.device:
        return lp
    cache = getattr(param, "_lowp_cache", None)
    if cache is not None and cache[0] == param._version and cache[1].dtype == dtype and cache[1].device == param.device:
        return cache[1]
    t = param.detach().to(dtype)
    try:
        param._lowp_cache = (param._version, t)
    except Exception:
        pass
    return t


# ----------------------------------------------------------------------------- augmentation / LM fusion
def specaugment(x, f_start, f_width, t_start, t_width, mask_value: float = 0.0):
    """Copy of ``x`` [B, F, T] with the frequency rows ``[f_start, f_start + f_width)`` and the time ranges
    ``[t_start, t_start + t_width)`` of every utterance set to ``mask_value`` (start / width: integer [B, n] or None)."""
    if _use_native(x) and x.dtype in (torch.float32, torch.bfloat16) and (t_start is None or t_start.shape[1] <= 32):
        i32 = lambda t: None if t is None else t.to(torch.int32).contiguous()  # noqa: E731
        return _nat().specaugment_(x.clone(memory_format=torch.contiguous_format), i32(f_start), i32(f_width), i32(t_start),
                                   i32(t_width), mask_value)
    return reference.specaugment(x, f_start, f_width, t_start, t_width, mask_value)


def ngram_advance(states, arc_keys, arc_w, arc_to, backoff_w, backoff_to, V: int, depth: int, default_score: float, start_state: int):
    if _use_native(states) and depth <= 16:
        return _nat().ngram_advance(states.contiguous(), arc_keys, arc_w, arc_to, backoff_w, backoff_to, V, depth, default_score,
                                    start_state)
    return reference.ngram_advance(states, arc_keys, arc_w, arc_to, backoff_w, backoff_to, V, depth, default_score, start_state)


# ----------------------------------------------------------------------------- dense layers
def linear(x, weight, bias=None, act: Optional[str] = None, residual=None, alpha: float = 1.0, dropout_p: float = 0.0):
    """``residual + alpha * dropout(act(x W^T + b))``; ``dropout_p`` > 0 means "apply dropout now" (callers pass 0 in eval)."""
    if _use_native(x) and x.dtype == torch.bfloat16:
        return _nat().linear(x, weight, bias, act, residual, alpha, dropout_p)
    return reference.linear(x, weight, bias, act, residual, alpha, dropout_p)


def layer_norm(x, weight, bias, eps: float = 1e-5):
    if _use_native(x) and x.dtype == torch.bfloat16:
        return _nat().layer_norm(x, weight, bias, eps)
    return reference.layer_norm(x, weight, bias, eps)


def relpos_attention(q, k, v, p, pos_bias_u, pos_bias_v, mask=None, dropout_p: float = 0.0, training: bool = False,
                     qkv=None):
    if _use_native(q) and q.dtype == torch.bfloat16:
        return _nat().relpos_attention(q, k, v, p, pos_bias_u, pos_bias_v, mask, dropout_p, training, qkv=qkv)
    return reference.relpos_attention(q, k, v, p, pos_bias_u, pos_bias_v, mask, dropout_p, training)


def mha_attention(q, k, v, mask=None, dropout_p: float = 0.0, training: bool = False, scale=None):
    if _use_native(q) and q.dtype == torch.bfloat16:
        return _nat().mha_attention(q, k, v, mask, scale, dropout_p, training)
    return reference.mha_attention(q, k, v, mask, dropout_p, training, scale)


def cross_attention(q, k, v, key_lengths=None, key_mask=None, scale: Optional[float] = None):
    """Attention of a decoder over an encoder's states, without the score matrix in memory: ``[B, Tq, H * D]``.

    ``q [B, Tq, H, D]``; ``k``, ``v [M, Tk, Hk, D]`` (any strides, e.g. slices of one fused projection).  ``B`` is a multiple of
    ``M``: query row ``b`` reads memory ``b // (B / M)``, so beams or sampled answers of one utterance share its states without
    copies; ``H`` is a multiple of ``Hk`` and head ``h`` reads key head ``h // (H / Hk)``.  Gradients of shared keys and values are
    summed over everything that read them.  ``key_lengths [M]`` (integers) hides the keys from a length on, ``key_mask [M, Tk]``
    (bool, True = hidden) single keys; both may be given.  A hidden place has no influence whatever it holds, and a query that sees
    no key gets zeros.  ``scale`` defaults to ``1 / sqrt(D)``.  No dropout on the weights: :func:`mha_attention` has it.

    On GPUs bf16 and fp16 with ``D`` a multiple of 8 up to 128 run as fused kernels, one for a few query rows per key head (decoding
    steps) and one for many; anything else runs the plain form, forward-mode differentiation too.  First derivatives only."""
    reference.check_cross_attention(q, k, v, key_lengths, key_mask)
    if _use_native(q) and q.dtype in (torch.bfloat16, torch.float16):
        return _nat().cross_attention(q, k, v, key_lengths, key_mask, scale)
    return reference.cross_attention(q, k, v, key_lengths, key_mask, scale)


def shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, prefix_lengths=None, scale: Optional[float] = None):
    """Decoding-step attention of a batch in which groups of rows share a prompt: ``[B, Tq, H * D]``.

    ``q [B, Tq, H, D]`` holds the newest ``Tq`` tokens of every row (their keys are in the cache already); ``k_prefix``,
    ``v_prefix [P, S, Hk, D]`` the prompts, row ``b`` continuing prompt ``b // (B / P)``, of which the first ``prefix_lengths [P]``
    positions count (default: all); ``k``, ``v [B, Smax, Hk, D]`` the rows' own caches, in which row ``b`` holds ``lengths[b]``
    positions, the new tokens included.  Token ``t`` sees its prompt and its row's positions up to its own, ``lengths[b] - Tq + t``;
    one that sees nothing gets zeros.  Lengths beyond a cache count as its size.  What stands behind the lengths has no influence;
    the new tokens' own keys and values are taken to be finite (an infinite value of a later one makes NaN of the earlier ones that share a
    call with it).  The prompt's keys and values are read once for the whole group.  Caches may have any strides (``[B, Hk, Smax, D]`` caches are passed as ``cache.transpose(1, 2)``).

    For inference: on GPUs there is no backward pass, and inputs that need gradients, of either mode, are refused."""
    reference.check_shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, prefix_lengths)
    if _use_native(q) and q.dtype in (torch.bfloat16, torch.float16):
        return _nat().shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, prefix_lengths, scale)
    return reference.shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, prefix_lengths, scale)


def conv_module_core(g, dw_weight, dw_bias, norm_type, norm_weight, norm_bias, running_mean, running_var,
                     pad_mask=None, training=False, momentum=0.1, eps=1e-5, left_pad=4, right_pad=4, cache=None,
                     cache_drop_size=0, bn_stats_reduce=None):
    if _use_native(g) and g.dtype == torch.bfloat16 and cache is None and norm_type in ("batch_norm", "layer_norm"):
        return _nat().conv_module_core(g, dw_weight, dw_bias, norm_type, norm_weight, norm_bias, running_mean,
                                         running_var, pad_mask, training, momentum, eps, left_pad, right_pad,
                                         bn_stats_reduce)
    return reference.conv_module_core(g, dw_weight, dw_bias, norm_type, norm_weight, norm_bias, running_mean,
                                      running_var, pad_mask, training, momentum, eps, left_pad, right_pad, cache,
                                      cache_drop_size, bn_stats_reduce)


def conformer_layer(layer, x, att_mask=None, pos_emb=None, pad_mask=None):
    """Whole Conformer layer (forward and backward each issued by one native call); ``None`` when the layer's configuration
    or this call is outside the executor's envelope and the caller should run the per-op path."""
    if not _use_native(x) or x.dtype != torch.bfloat16:
        return None
    from . import native_layer

    return native_layer.conformer_layer(layer, x, att_mask, pos_emb, pad_mask)


def lstm(x, weights, h0=None, c0=None, num_layers=1, dropout=0.0, training=False):
    if _use_native(x) and x.dtype == torch.bfloat16 and not (dropout > 0 and training) and hasattr(_nat(), "lstm"):
        return _nat().lstm(x, weights, h0, c0, num_layers)
    return reference.lstm(x, weights, h0, c0, num_layers, dropout, training)


# ----------------------------------------------------------------------------- losses
def transducer_joint_loss(f, g, w, b, targets, f_len, y_len, blank, durations, sigma, act="relu",
                          fastemit_lambda=0.0, sub_batch=0, dropout_p: float = 0.0):
    if _use_native(f) and f.dtype == torch.bfloat16 and act == "relu":
        return _nat().transducer_joint_loss(f, g, w, b, targets, f_len, y_len, blank, durations, sigma,
                                              fastemit_lambda, dropout_p)
    return reference.transducer_joint_loss(f, g, w, b, targets, f_len, y_len, blank, durations, sigma, act,
                                           fastemit_lambda, sub_batch, dropout_p=dropout_p)


def transducer_loss_from_logits(logits, targets, f_len, y_len, blank, durations, sigma=0.0):
    if _use_native(logits):
        return _nat().transducer_loss_from_logits(logits, targets, f_len, y_len, blank, durations, sigma)
    return reference.tdt_loss_from_logits(logits, targets, f_len, y_len, blank, durations, sigma)


def ctc_loss(log_probs, targets, input_lengths, target_lengths, blank, zero_infinity=True):
    if _use_native(log_probs) and hasattr(_nat(), "ctc_loss"):
        return _nat().ctc_loss(log_probs, targets, input_lengths, target_lengths, blank)
    return reference.ctc_loss(log_probs, targets, input_lengths, target_lengths, blank, zero_infinity)


def policy_loss(logits, targets, mask, old_logp, advantages, ref_logp=None, clip: float = 0.2, clip_high: Optional[float] = None,
                kl_beta: float = 0.0):
    """Clipped policy loss with a KL term, straight from logits: ``(loss, logp)``.

    ``logits [N, T, V]`` or ``[N, T, C, V]`` (C codebooks), ``targets`` the sampled tokens ``[N, T(, C)]``, ``mask [N, T]`` non-zero at
    positions that count (None: all), ``old_logp`` the log-probabilities under the policy that sampled, ``ref_logp`` those under the
    frozen policy (with ``kl_beta`` > 0), both of the targets' shape, ``advantages [N]``.  With ``r = exp(logp - old_logp)`` a position's
    term is ``-min(r A, clip(r, 1 - clip, 1 + clip_high) A) + kl_beta (exp(d) - d - 1)``, ``d = ref_logp - logp``; the loss is the mean
    over all counted positions (0 when there are none).  ``logp`` (fp32, detached, 0 where masked) is the next ``old_logp``.  Gradients
    go to ``logits`` only.  Masked positions are not read, whatever they hold.  On GPUs a counted target outside the vocabulary makes
    the loss NaN (the CPU raises), and a forward pass that needs gradients holds the logits' gradient until backward."""
    reference.check_sequence_loss("policy_loss", logits, targets, mask, (("old_logp", old_logp), ("ref_logp", ref_logp)),
                                  (("advantages", advantages, logits.shape[0] if logits.dim() > 0 else 0),))
    if kl_beta != 0.0 and ref_logp is None:
        raise ValueError("a KL term (kl_beta != 0) needs ref_logp")
    if clip < 0 or (clip_high is not None and clip_high < 0):
        raise ValueError(f"clip ranges must not be negative, got {clip}, {clip_high}")
    if _use_native(logits) and logits.dtype in (torch.bfloat16, torch.float16, torch.float32) and targets.numel() > 0:
        return _nat().policy_loss(logits, targets, mask, old_logp, advantages, ref_logp, clip, clip_high, kl_beta)
    return reference.policy_loss(logits, targets, mask, old_logp, advantages, ref_logp, clip, clip_high, kl_beta)


def preference_loss(logits, targets, mask, ref_logp, beta: float = 0.1, loss_type: str = "dpo", reward_gap=None):
    """Paired preference loss straight from logits: ``(loss, rewards)``.

    The first half of the ``2 N`` sequences holds the chosen answers, the second half the rejected ones in the same order; ``logits``,
    ``targets``, ``mask`` and ``ref_logp`` as in :func:`policy_loss`.  With ``ratio`` the sum of ``logp - ref_logp`` over a sequence's
    counted positions and ``margin = ratio_chosen - ratio_rejected``, a pair's loss is ``-log sigmoid(beta margin)`` (``dpo``),
    ``(margin - 1 / (2 beta))^2`` (``ipo``) or ``(beta margin - reward_gap)^2`` (``rpo_sq``, ``reward_gap [N]``); the loss is their mean.
    ``rewards [2 N]`` = ``beta * ratio`` (fp32, detached)."""
    N = logits.shape[0] if logits.dim() > 0 else 0
    reference.check_sequence_loss("preference_loss", logits, targets, mask, (("ref_logp", ref_logp),), (("reward_gap", reward_gap, N // 2),))
    if N == 0 or N % 2:
        raise ValueError(f"preference_loss takes pairs: chosen answers, then as many rejected ones; got {N} sequences")
    if loss_type not in ("dpo", "ipo", "rpo_sq"):
        raise NotImplementedError(f"loss type {loss_type} is not implemented")
    if loss_type == "rpo_sq" and reward_gap is None:
        raise ValueError("rpo_sq needs the reward gap of every pair")
    if loss_type == "ipo" and beta == 0.0:
        raise ValueError("ipo aims at a margin of 1 / (2 beta): beta must not be zero")
    if _use_native(logits) and logits.dtype in (torch.bfloat16, torch.float16, torch.float32) and targets.numel() > 0:
        return _nat().preference_loss(logits, targets, mask, ref_logp, beta, loss_type, reward_gap)
    return reference.preference_loss(logits, targets, mask, ref_logp, beta, loss_type, reward_gap)


# ----------------------------------------------------------------------------- front-end
def logmel(x, seq_len, window, fb, n_fft, hop, win_length, preemph=0.97, mag_power=2.0, log_zero_guard=2 ** -24,
           normalize="per_feature", pad_to=0, pad_value=0.0, dither=0.0, log=True):
    if _use_native(x) and normalize in ("per_feature", None) and mag_power == 2.0 and log and n_fft == 512 and hasattr(_nat(), "logmel"):
        return _nat().logmel(x, seq_len, window, fb, n_fft, hop, win_length, preemph, log_zero_guard,
                               normalize, pad_to, pad_value, dither)
    return reference.logmel(x, seq_len, window, fb, n_fft, hop, win_length, preemph, mag_power, log_zero_guard,
                            normalize, pad_to, pad_value, dither, log=log)


# ----------------------------------------------------------------------------- optimizer
def adamw_flat(master, grad, exp_avg, exp_avg_sq, lowp, lr, beta1, beta2, eps, weight_decay, step, scalars):
    """One fused AdamW pass; ``scalars[1]`` (device memory) holds the gradient multiplier (clip x scale)."""
    if _use_native(master):
        return _nat().adamw_flat(master, grad, exp_avg, exp_avg_sq, lowp, lr, beta1, beta2, eps, weight_decay, step,
                                   scalars)
    return reference.adamw_flat(master, grad, exp_avg, exp_avg_sq, lowp, lr, beta1, beta2, eps, weight_decay, step,
                                clip_coef=scalars[1])


def grad_norm_clip_coef(flat_grad, scalars, max_norm: float, grad_scale: float = 1.0):
    """scalars[0] <- ||grad * grad_scale||_2, scalars[1] <- grad_scale * min(1, max_norm / (norm + 1e-6))."""
    if _use_native(flat_grad):
        return _nat().grad_norm_clip_coef(flat_grad, scalars, max_norm, grad_scale)
    norm = flat_grad.float().norm() * grad_scale
    scalars[0] = norm
    scalars[1] = grad_scale * torch.clamp(max_norm / (norm + 1e-6), max=1.0)


from . import native  # noqa: E402,F401  (binding module; the shared library itself is loaded on first use)
