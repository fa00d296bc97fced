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
hold. A counted position whose target lies outside [0, V) has the log-probability NaN.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

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
    _lib.same_device(logits, targets=targets, mask=mask)
    return targets.to(torch.long).contiguous(), _per_token("mask", mask, targets)


def _per_token(name, t, targets):
    """t, broadcast to the targets' shape, contiguous (None stays None)."""
    if t is None:
        return None
    try:
        return t.detach().expand(targets.shape).resolve_neg().contiguous()
    except RuntimeError:
        raise ValueError(f"{name} {tuple(t.shape)} does not broadcast to the targets "
                         f"{tuple(targets.shape)}") from None


def _floats(name, t, targets):
    if t is None:
        return None
    _lib.require_device(t)
    _lib.same_device(targets, **{name: t})
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, got {t.dtype}")
    return _per_token(name, t.to(torch.float32), targets)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _layout(logits):
    """(logits as read, the arguments that describe them to the library)."""
    t, rows, inner, so, si = _rows(logits)
    return t, (_lib.DTYPE_CODE[t.dtype], rows, inner, t.shape[-1], so, si)


def _grad(ctx, saved, coef, per, scale0, scale1):
    """The logits' gradient from what the forward saved."""
    logits, targets, mask, stats = saved
    dev = coef.device
    logits = logits.to(device=dev, dtype=ctx.dtype)
    back = lambda t, dt: None if t is None else _lib.dense(t.to(device=dev, dtype=dt))  # noqa: E731
    targets, mask, stats = back(targets, torch.long), back(mask, torch.bool), back(stats, torch.float32)
    t, args = _layout(logits)
    grad = torch.empty(logits.shape, dtype=t.dtype, device=dev)
    with _lib.device_of(t):
        _lib.check(_lib.lib().lema_token_logprobs_grad(
            t.data_ptr(), *args, targets.data_ptr(), _ptr(mask), ctx.temperature, stats.data_ptr(),
            coef.data_ptr(), per, _ptr(scale0), _ptr(scale1), grad.data_ptr(), _lib.stream_of(t)))
    return grad


def _logprobs(logits, targets, mask, temperature, want_stats, want_64=False):
    """(lp, lp in 64 bits or None, stats or None)."""
    t, args = _layout(logits)
    lp = t.new_empty(targets.shape, dtype=torch.float32)
    lp64 = t.new_empty(targets.shape, dtype=torch.float64) if want_64 else None
    stats = t.new_empty(targets.shape + (2,), dtype=torch.float32) if want_stats else None
    with _lib.device_of(t):
        _lib.check(_lib.lib().lema_token_logprobs(
            t.data_ptr(), *args, targets.data_ptr(), _ptr(mask), temperature, lp.data_ptr(), _ptr(lp64),
            _ptr(stats), _lib.stream_of(t)))
    return lp, lp64, stats


def _remember(ctx, logits, targets, mask, stats, temperature, *more):
    ctx.save_for_backward(logits, targets, mask, stats, *more)
    ctx.dtype, ctx.temperature = logits.dtype, temperature


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature):
        lp, _, stats = _logprobs(logits, targets, mask, temperature, True)
        _remember(ctx, logits, targets, mask, stats, temperature)
        return lp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return _grad(ctx, ctx.saved_tensors, _lib.dense(g), 1, None, None), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, mask: torch.Tensor | None = None,
                   temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / temperature) at the targets: logits [..., V], targets [...], fp32 out;
    the log-probabilities that policy_loss and preference_loss take of the policy that sampled an
    answer, and of the reference. One read of the logits, and one more read and a write for
    their gradient."""
    targets, mask = _check(logits, targets, mask, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobs.apply(logits, targets, mask, float(temperature))
    return _logprobs(logits, targets, mask, float(temperature), False)[0]


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature, old, adv, ref, low, high, kl):
        t, args = _layout(logits)
        f32 = lambda *shape: t.new_empty(shape, dtype=torch.float32)  # noqa: E731
        lp, stats, loss, inv_n = f32(*targets.shape), f32(*targets.shape, 2), f32(), f32()
        term, coef = f32(targets.numel()), f32(targets.numel())
        with _lib.device_of(t):
            _lib.check(_lib.lib().lema_policy_loss(
                t.data_ptr(), *args, targets.data_ptr(), _ptr(mask), temperature, old.data_ptr(),
                adv.data_ptr(), _ptr(ref), low, high, kl, lp.data_ptr(), stats.data_ptr(),
                term.data_ptr(), coef.data_ptr(), loss.data_ptr(), inv_n.data_ptr(), _lib.stream_of(t)))
        _remember(ctx, logits, targets, mask, stats, temperature, coef, inv_n)
        ctx.mark_non_differentiable(lp)
        ctx.set_materialize_grads(False)
        return loss, lp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 10
        *saved, coef, inv_n = ctx.saved_tensors
        coef, inv_n = (_lib.dense(t.to(device=g.device, dtype=torch.float32)) for t in (coef, inv_n))
        return (_grad(ctx, saved, coef, 1, _lib.dense(g), inv_n),) + (None,) * 9


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                advantages: torch.Tensor, ref_logprobs: torch.Tensor | None = None,
                mask: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_weight: float = 0.0, temperature: float = 1.0) -> PolicyLoss:
    """The mean over the counted positions of

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_weight (e^g - g - 1)

    with lp = token_logprobs(logits, targets), r = e^(lp - old_logprobs), A = advantages and
    g = ref_logprobs - lp; 0 where the mask counts nothing. old_logprobs, advantages, ref_logprobs
    and mask broadcast to the targets' shape ([B, 1] advantages give each answer one)."""
    targets, mask = _check(logits, targets, mask, temperature)
    old, adv, ref = (_floats(n, t, targets) for n, t in
                     (("old_logprobs", old_logprobs), ("advantages", advantages),
                      ("ref_logprobs", ref_logprobs)))
    if old is None or adv is None:
        raise TypeError("old_logprobs and advantages are needed")
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"clip distances must not be negative, got {clip_low} and {clip_high}")
    if kl_weight != 0 and ref is None:
        raise ValueError("kl_weight needs ref_logprobs")
    return PolicyLoss(*_PolicyLoss.apply(logits, targets, mask, float(temperature), old, adv, ref,
                                         float(clip_low), float(clip_high), float(kl_weight)))


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature, ref, beta, smooth):
        N, T = targets.shape
        lp, lp64, stats = _logprobs(logits, targets, mask, temperature, True, want_64=True)
        loss, margins, coef = (lp.new_empty(s) for s in ((), (N // 2,), (N,)))
        with _lib.device_of(lp):
            _lib.check(_lib.lib().lema_preference_loss(
                lp64.data_ptr(), ref.data_ptr(), _ptr(mask), N // 2, T, beta, smooth, loss.data_ptr(),
                margins.data_ptr(), coef.data_ptr(), _lib.stream_of(lp)))
        _remember(ctx, logits, targets, mask, stats, temperature, coef)
        ctx.mark_non_differentiable(margins, lp)
        ctx.set_materialize_grads(False)
        return loss, margins, lp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        if g is None:
            return (None,) * 7
        *saved, coef = ctx.saved_tensors
        coef = _lib.dense(coef.to(device=g.device, dtype=torch.float32))
        T = saved[1].shape[1]
        return (_grad(ctx, saved, coef, max(1, T), _lib.dense(g), None),) + (None,) * 6


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor,
                    mask: torch.Tensor | None = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, temperature: float = 1.0) -> PreferenceLoss:
    """The paired preference loss of 2 P answers of T tokens, logits [2 P, T, V]: answer p of the
    first P is preferred to answer P + p. With s an answer's sum of lp - ref_logprobs over its
    counted positions and m = beta (s_chosen - s_rejected), the mean over the pairs of
    -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m). ref_logprobs and mask
    broadcast to the targets' shape [2 P, T]. The sums are formed in 64 bits."""
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
