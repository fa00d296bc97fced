"""Losses of a hard-mode model's answers, from logits, with their gradients in HIP.

    token_logprobs(logits, targets)          log-probabilities of given tokens
    policy_loss(logits, targets, ...)        clipped policy loss with a KL term to a reference
    preference_loss(logits, targets, ...)    paired preference loss on chosen and rejected answers

The reference trains on next-token cross-entropy only (code/lema/train.py:131-152, here
`model.lm_loss`); these are what fine-tuning on sampled answers adds (LemaDecoder samples
them). Logits are float32, float16 or bfloat16 on the device, [..., V] with a contiguous last dim
(other layouts are copied; a slice like logits[:, :-1] is read in place); log-probabilities and
losses are fp32. Only the logits are differentiable. A position that `mask` leaves out is not
read: its log-probability and gradient are zero whatever its logits, target and other inputs
hold. A counted position whose target lies outside [0, V) has the log-probability NaN, and the
gradient NaN unless its log-probability's gradient is zero. Logits of
-inf have the probability 0; one whose distance to its row's maximum leaves fp32's range may too.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

__all__ = ["token_logprobs", "policy_loss", "preference_loss", "PolicyLoss", "PreferenceLoss"]


class PolicyLoss(NamedTuple):
    loss: torch.Tensor        # fp32 scalar, differentiable in the logits
    logprobs: torch.Tensor    # fp32, like the targets; no gradient


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor        # fp32 scalar, differentiable in the logits
    margins: torch.Tensor     # fp32 [pairs], beta times the pair's difference; no gradient
    logprobs: torch.Tensor    # fp32, like the targets; no gradient


def _rows(logits: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """logits, their rows, and how the rows lie: (rows per outer step, outer and inner stride).
    Copies only where the rows do not fit two strides."""
    V = logits.shape[-1]
    rows = logits.numel() // V
    t = logits.resolve_neg()
    if rows == 0:
        return t, 0, 1, 0, V
    if V > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    # dims of more than one step, outermost first, merged where they are laid out as one
    dims: list[tuple[int, int]] = []
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = (dims[-1][0] * n, s)
        else:
            dims.append((n, s))
    if len(dims) > 2:
        t, dims = t.contiguous(), [(rows, V)]
    if len(dims) == 2:
        return t, rows, dims[1][0], dims[0][1], dims[1][1]
    return t, rows, rows, 0, dims[0][1] if dims else V


def _check(logits, targets, mask, temperature):
    """The arguments every loss takes, as the kernels read them: (targets, mask)."""
    if not (logits.is_cuda and targets.is_cuda):
        _lib.require_device(logits, targets)
    if logits.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if targets.dtype not in (torch.long, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    if logits.dim() < 1 or logits.shape[:-1] != targets.shape:
        raise ValueError(f"logits {tuple(logits.shape)} do not match targets {tuple(targets.shape)}")
    if logits.shape[-1] < 1:
        raise ValueError("logits over an empty vocabulary")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"the temperature must be positive, got {temperature}")
    if mask is not None and mask.dtype != torch.bool:
        raise TypeError(f"the mask must be bool, got {mask.dtype}")
    if targets.device != logits.device or (mask is not None and mask.device != logits.device):
        _lib.same_device(logits, targets=targets, mask=mask)
    return targets.long().contiguous(), _per_token("mask", mask, targets)


def _per_token(name, t, targets):
    """t, broadcast to the targets' shape, contiguous (None stays None)."""
    if t is None:
        return None
    if t.shape == targets.shape:
        return _lib.dense(t)
    try:
        return _lib.dense(t.expand(targets.shape))
    except RuntimeError:
        raise ValueError(f"{name} {tuple(t.shape)} does not broadcast to the targets "
                         f"{tuple(targets.shape)}") from None


def _floats(name, t, targets):
    if t is None:
        return None
    if (t.dtype is torch.float32 and t.shape == targets.shape and t.device == targets.device
            and t.is_contiguous() and not t.is_neg()):
        return t
    if t.device != targets.device:
        _lib.require_device(t)
        _lib.same_device(targets, **{name: t})
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, got {t.dtype}")
    return _per_token(name, t.detach().float(), targets)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _layout(logits):
    """(logits as read, the arguments that describe them to the library)."""
    t, rows, inner, so, si = _rows(logits)
    return t, (_lib.DTYPE_CODE[t.dtype], rows, inner, t.shape[-1], so, si)


# What a forward leaves for its backward is one fp32 tensor: (max, 1 / sum) of each row, then the
# coefficients (of each row for the policy loss, of each answer for the preference loss), then for
# the policy loss 1 / the counted rows, and room for the rows' terms.

def _remember(ctx, logits, t, args, targets, mask, state, temperature):
    ctx.save_for_backward(logits, targets, mask, state)
    # the description holds for the saved logits unless they were copied to be read
    ctx.logits = (t.data_ptr(), t.stride(), args) if t is logits else None
    ctx.dtype, ctx.temperature = logits.dtype, temperature
    ctx.set_materialize_grads(False)


def _grad(ctx, like, coef, per, scale0, inv_n, grad=None):
    """The logits' gradient from what the forward saved. coef: a tensor, or None for the state's;
    inv_n: whether the state has it; grad: the one that the forward wrote for scale0 = 1."""
    logits, targets, mask, state = ctx.saved_tensors
    dev = like.device
    if logits.dtype is not ctx.dtype or logits.device != dev:
        logits = logits.to(device=dev, dtype=ctx.dtype)
    targets, state = _lib.saved(targets, like, torch.long), _lib.saved(state, like, torch.float32, 8)
    mask = _lib.saved(mask, like, torch.bool) if mask is not None else None
    if ctx.logits is not None and ctx.logits[:2] == (logits.data_ptr(), logits.stride()):
        t, args = logits, ctx.logits[2]
    else:
        t, args = _layout(logits)
    at, rows = state.data_ptr(), args[1]
    out = grad if grad is not None else torch.empty(logits.shape, dtype=t.dtype, device=dev)
    with _lib.device_of(like):
        _lib.check(_lib.lib().lema_token_logprobs_grad(
            t.data_ptr(), *args, targets.data_ptr(), _ptr(mask), ctx.temperature, at,
            coef.data_ptr() if coef is not None else at + 8 * rows, per, _ptr(scale0),
            at + 12 * rows if inv_n else None, grad is not None, out.data_ptr(), _lib.stream_of(like)))
    return out


def _logprobs(t, args, targets, mask, temperature, stats=None, lp64=None):
    lp = t.new_empty(targets.shape, dtype=torch.float32)
    with _lib.device_of(t):
        _lib.check(_lib.lib().lema_token_logprobs(
            t.data_ptr(), *args, targets.data_ptr(), _ptr(mask), temperature, lp.data_ptr(), _ptr(lp64),
            _ptr(stats), _lib.stream_of(t)))
    return lp


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature):
        t, args = _layout(logits)
        state = t.new_empty(2 * args[1], dtype=torch.float32)
        lp = _logprobs(t, args, targets, mask, temperature, state)
        _remember(ctx, logits, t, args, targets, mask, state, temperature)
        return lp

    @staticmethod
    @_lib.once
    def backward(ctx, g):
        if g is None:
            return (None,) * 4
        g = _lib.dense(g)
        return _grad(ctx, g, g, 1, None, False), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, mask: torch.Tensor | None = None,
                   temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / temperature) at the targets: logits [..., V], targets [...], fp32 out;
    the log-probabilities that policy_loss and preference_loss take of the policy that sampled an
    answer, and of the reference. One read of the logits, and one more read and a write for
    their gradient."""
    targets, mask = _check(logits, targets, mask, temperature)
    if _lib.needs_grad(logits):
        return _TokenLogprobs.apply(logits, targets, mask, float(temperature))
    return _logprobs(*_layout(logits), targets, mask, float(temperature))


class _PolicyLoss(torch.autograd.Function):
    """The forward writes the gradient too, for a gradient of 1 of the loss, while it holds a row's
    logits: a batch's logits do not fit a cache, and reading them again would be a third of the
    traffic. The first backward hands that tensor out, computed anew where the loss's gradient
    is not 1. A second one computes its own, and so does one that is not recorded into the graph
    that the forward was (its replays would not write the tensor again)."""

    @staticmethod
    def forward(ctx, logits, targets, mask, temperature, old, adv, ref, low, high, kl, scale, want_grad):
        t, args = _layout(logits)
        n = args[1]
        lp, loss = t.new_empty(targets.shape, dtype=torch.float32), t.new_empty((), dtype=torch.float32)
        state = t.new_empty(4 * n + 1, dtype=torch.float32)
        stream = _lib.stream_of(t)
        at = state.data_ptr()
        with _lib.device_of(t):
            ctx.capture = _lib.lib().lema_capture_id(stream)
            ctx.grad = (torch.empty(logits.shape, dtype=t.dtype, device=t.device)
                        if want_grad and ctx.capture >= 0 else None)
            _lib.check(_lib.lib().lema_policy_loss(
                t.data_ptr(), *args, targets.data_ptr(), _ptr(mask), temperature, old.data_ptr(),
                adv.data_ptr(), _ptr(ref), low, high, kl, scale, lp.data_ptr(), at, at + 12 * n + 4, at + 8 * n,
                loss.data_ptr(), at + 12 * n, _ptr(ctx.grad), stream))
        _remember(ctx, logits, t, args, targets, mask, state, temperature)
        ctx.mark_non_differentiable(lp)
        return loss, lp

    @staticmethod
    @_lib.once
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 12
        g = _lib.dense(g)
        grad = ctx.__dict__.pop("grad", None)
        if grad is not None and _lib.lib().lema_capture_id(_lib.stream_of(g)) != ctx.capture:
            grad = None
        return (_grad(ctx, g, None, 1, g, True, grad),) + (None,) * 11


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                advantages: torch.Tensor, ref_logprobs: torch.Tensor | None = None,
                mask: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_weight: float = 0.0, temperature: float = 1.0, scale: float = 1.0) -> PolicyLoss:
    """`scale` times the mean over the counted positions of

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_weight (e^g - g - 1)

    with lp = token_logprobs(logits, targets), r = e^(lp - old_logprobs), A = advantages and
    g = ref_logprobs - lp; 0 where the mask counts nothing. old_logprobs, advantages, ref_logprobs
    and mask broadcast to the targets' shape ([B, 1] advantages give each answer one).

    The forward already writes the logits' gradient for a gradient of 1 of the loss. A factor that
    the loss is to have (one over the steps that gradients are accumulated for) is best given as
    `scale`: multiplied afterwards, it makes the backward read the logits again."""
    targets, mask = _check(logits, targets, mask, temperature)
    old, adv, ref = (_floats(n, t, targets) for n, t in
                     (("old_logprobs", old_logprobs), ("advantages", advantages),
                      ("ref_logprobs", ref_logprobs)))
    if old is None or adv is None:
        raise TypeError("old_logprobs and advantages are needed")
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"clip distances must not be negative, got {clip_low} and {clip_high}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be a number, got {scale}")
    if kl_weight != 0 and ref is None:
        raise ValueError("kl_weight needs ref_logprobs")
    want = torch.is_grad_enabled() and logits.requires_grad
    return PolicyLoss(*_PolicyLoss.apply(logits, targets, mask, float(temperature), old, adv, ref,
                                         float(clip_low), float(clip_high), float(kl_weight), float(scale), want))


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature, ref, beta, smooth):
        t, args = _layout(logits)
        N, T = targets.shape
        state = t.new_empty(2 * N * T + N, dtype=torch.float32)
        lp64 = t.new_empty(targets.shape, dtype=torch.float64)
        lp = _logprobs(t, args, targets, mask, temperature, state, lp64)
        loss, margins = lp.new_empty(()), lp.new_empty(N // 2)
        with _lib.device_of(t):
            _lib.check(_lib.lib().lema_preference_loss(
                lp64.data_ptr(), ref.data_ptr(), _ptr(mask), N // 2, T, beta, smooth, loss.data_ptr(),
                margins.data_ptr(), state.data_ptr() + 8 * N * T, _lib.stream_of(t)))
        _remember(ctx, logits, t, args, targets, mask, state, temperature)
        ctx.per = max(1, T)
        ctx.mark_non_differentiable(margins, lp)
        return loss, margins, lp

    @staticmethod
    @_lib.once
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 7
        g = _lib.dense(g)
        return (_grad(ctx, g, None, ctx.per, g, False),) + (None,) * 6


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor,
                    mask: torch.Tensor | None = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, temperature: float = 1.0) -> PreferenceLoss:
    """The paired preference loss of 2 P answers of T tokens, logits [2 P, T, V]: answer p of the
    first P is preferred to answer P + p. With s an answer's sum of lp - ref_logprobs over its
    counted positions and m = beta (s_chosen - s_rejected), the mean over the pairs of
    -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m), where a part of weight 0
    is left out. ref_logprobs and mask broadcast to the targets' shape [2 P, T]. The sums are formed
    in 64 bits."""
    targets, mask = _check(logits, targets, mask, temperature)
    if targets.dim() != 2 or targets.shape[0] % 2 or targets.shape[0] == 0:
        raise ValueError(f"targets must be [2 P, T] with P >= 1, got {tuple(targets.shape)}")
    ref = _floats("ref_logprobs", ref_logprobs, targets)
    if ref is None:
        raise TypeError("ref_logprobs are needed")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"label_smoothing must lie in [0, 1], got {label_smoothing}")
    if not math.isfinite(beta):
        raise ValueError(f"beta must be a number, got {beta}")
    return PreferenceLoss(*_PreferenceLoss.apply(logits, targets, mask, float(temperature), ref,
                                                 float(beta), float(label_smoothing)))
