"""The LEMA transformer on MI355X: the reference's `ModelConfig` / `Transformer`
(code/lema/model.py) for an all-LEMA model in hard mode, the configuration in which the
exact op runs and a retrieval cache can be attached.

Pre-RMSNorm, SwiGLU MLP, untied head, no biases, no positional encoding
(code/lema/model.py:1-9). The projections, MLP and head are bf16 (or fp32) GEMMs on the
matrix cores through torch; the attention of every block is the exact op of this package
(sign-pack, latest-match resolve and gather in HIP), and a cached forward exchanges each
layer's codes against the HBM store with no host round trip.

Parameters are created and initialised in the reference's module order (embedding, then per
block norm1, q, k, v, o, norm2, gate, up, down, then norm_f, lm_head; Gaussian std
1/sqrt(fan_in) for every Linear and 1/sqrt(dim) for the embedding, the two residual-branch
outputs scaled by 1/sqrt(2 * depth): code/lema/model.py:258-281), so the same seed gives the
same weights.

Forwards without a cache are differentiable where the exact op is (in the values, not in the
codes): the embedding, the norms, SwiGLU and the loss have hand-written gradients in bf16.

In bf16 on the GPU the SwiGLU product, both pre-norms (the MLP's with the attention residual
add), the final norm and the loss run as fused HIP kernels (the reference compiles these
segments with torch.compile). The norm kernel rounds like torch's RMSNorm (one rounding of
x * rstd * w from fp32) but adds up the mean of squares in its own order, so a rare element
of the attention input lands one bf16 ulp from torch's. The codes, the signs of that input's
projections, can then differ from the ones torch's norm gives, only at pre-activations
within 1e-3 of zero (the stated binarization tolerance; at the full LM shape 9 of 1e8 code
bits of the first layer).

Only the hard (exact) op is implemented: the training surrogate (stick-breaking relaxation,
straight-through binarization) and the softmax / gated-deltanet baselines are not part of the
exact-match path.
"""
from __future__ import annotations

import contextlib
import dataclasses
import math
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib, fp8
from .attention import _unwatched, code_dtype_for, lema_from_codes, lema_hard, pack_codes

__all__ = ["ModelConfig", "SwiGLU", "Attention", "Block", "Transformer", "lm_loss", "rms_norm",
           "layer_norm", "embed", "argmax_into", "load_trained",
           "swiglu", "gated_linear", "cross_entropy_sum"]

# ------------------------------------------------------------------ fused bf16 segments
# On the GPU in bf16 the SwiGLU product, the residual add with the next pre-norm, and the loss
# run as one HIP kernel each (liblema_hip.so); other dtypes and devices use the torch ops.

def _fused(*ts: torch.Tensor) -> bool:
    """Whether the kernels take the tensors as they lie: bf16 on the GPU, contiguous, from a 16-byte
    boundary on (a slice, or a parameter in a flat buffer, may start elsewhere). An 8-bit weight is none."""
    for t in ts:
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.bfloat16 and t.is_contiguous() and t.data_ptr() % 16 == 0):
            return False
    return True


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _norm_forward(x, d, w, b, eps, center):
    """h and s = x + d (None without d) of contiguous inputs, w's elements to a row."""
    D = w.numel() if isinstance(w, torch.Tensor) else w
    w = w if isinstance(w, torch.Tensor) else None
    h = torch.empty_like(x)
    s = torch.empty_like(x) if d is not None else None
    with _lib.device_of(x):
        if center:
            _lib.check(_lib.lib().lema_layer_norm(
                x.data_ptr(), _ptr(d), _ptr(w), _ptr(b), _lib.DTYPE_CODE[x.dtype], eps, x.numel() // D, D,
                _ptr(s), h.data_ptr(), _lib.stream_of(x)))
        else:
            _lib.check(_lib.lib().lema_rmsnorm_bf16(
                x.data_ptr(), _ptr(d), _ptr(w), eps, x.numel() // D, D, _ptr(s), h.data_ptr(),
                _lib.stream_of(x)))
    return h, s


class _Norm(torch.autograd.Function):
    """h, and s = x + d where d is given, with the gradients of x, d and the weights."""

    @staticmethod
    def forward(ctx, x, d, w, b, D, eps, center):
        h, s = _norm_forward(x, d, w if w is not None else D, b, eps, center)
        ctx.save_for_backward(x if s is None else s, w)
        ctx.norm = D, eps, int(center), d is not None, b is not None
        ctx.scratch = _lib.lib().lema_norm_grad_workspace_bytes(x.numel() // D, D)
        ctx.w_shape = w.shape if w is not None else b.shape if b is not None else None
        ctx.set_materialize_grads(False)
        return h if s is None else (h, s)

    @staticmethod
    @_lib.once
    def backward(ctx, gh, gs=None):
        D, eps, center, has_d, has_b = ctx.norm
        want_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        want_w, want_b = ctx.needs_input_grad[2:4]
        if gh is None:                                # only the sum was used
            return gs, gs, None, None, None, None, None
        s, w = ctx.saved_tensors
        gh = _lib.dense(gh)
        gs = _lib.dense(gs) if gs is not None else None
        s = _lib.saved(s, gh, gh.dtype)
        w = _lib.saved(w, gh, gh.dtype) if w is not None else None
        L = _lib.lib()
        gx = torch.empty_like(s) if want_x else None
        gw = gh.new_empty(ctx.w_shape) if want_w else None
        gb = gh.new_empty(ctx.w_shape) if want_b and has_b else None
        ws = gh.new_empty(ctx.scratch, dtype=torch.uint8) if want_w or want_b else None
        with _lib.device_of(gh):
            _lib.check(L.lema_norm_grad(
                s.data_ptr(), _ptr(w), gh.data_ptr(), _ptr(gs), _lib.DTYPE_CODE[gh.dtype], center, eps,
                s.numel() // D, D, _ptr(gx), _ptr(gw), _ptr(gb), _ptr(ws), ctx.scratch,
                _lib.stream_of(gh)))
        return gx, gx if has_d else None, gw, gb, None, None, None


def rms_norm(x: torch.Tensor, norm: nn.RMSNorm, d: torch.Tensor | None = None):
    """norm(x + d) and x + d (or norm(x), x when d is None), one pass in bf16; the gradients of
    x, d and the weight take one more and a sum over workgroups."""
    if not (norm.weight is not None and _fused(x, norm.weight) and norm.weight.shape == x.shape[-1:]
            and (d is None or _fused(d) and d.shape == x.shape)
            and x.shape[-1] % 8 == 0 and x.shape[-1] <= 4096):
        x = x if d is None else x + d
        return norm(x), x
    eps = float(norm.eps if norm.eps is not None else torch.finfo(x.dtype).eps)
    return _norm(x, d, norm.weight, None, x.shape[-1], eps, False)


def _norm(x, d, w, b, D, eps, center):
    """norm(x + d) and x + d of contiguous inputs that the kernels take, with or without a graph."""
    if _lib.needs_grad(x, d, w, b):
        out = _Norm.apply(x, d, w, b, D, eps, center)
        return out if d is not None else (out, x)
    h, s = _norm_forward(x, d, w if w is not None else D, b, eps, center)
    return h, s if d is not None else x


LAYER_NORM_MAX = 16384  # elements of a row that the kernels hold in registers


def layer_norm(x: torch.Tensor, norm: nn.LayerNorm, d: torch.Tensor | None = None):
    """norm(x + d) and x + d (or norm(x), x when d is None), as rms_norm for an nn.LayerNorm: one
    pass on the GPU in float32, float16 or bfloat16, the sum rounded to that type first, mean and
    variance in fp32 from the centred row. Differentiable in x, d, weight and bias. Rows of at
    most 16384 elements of any length and alignment; the parameters have x's type. On the CPU, and
    in float64, the torch operations."""
    if d is not None and d.shape != x.shape:
        raise ValueError(f"the addend {tuple(d.shape)} does not match x {tuple(x.shape)}")
    if not x.is_cuda or x.dtype not in _lib.DTYPE_CODE:
        x = x if d is None else x + d
        return norm(x), x
    dims, shape = norm.normalized_shape, x.shape
    if shape[len(shape) - len(dims):] != dims:
        raise ValueError(f"x {tuple(shape)} does not end in the norm's shape {tuple(dims)}")
    D = math.prod(dims)
    if not 1 <= D <= LAYER_NORM_MAX:
        raise ValueError(f"rows of {D} elements: layer_norm takes 1 to {LAYER_NORM_MAX}")
    w, b = norm.weight, norm.bias
    for name, t in (("the addend", d), ("the weight", w), ("the bias", b)):
        if t is not None and (t.dtype is not x.dtype or t.device != x.device):
            _lib.same_device(x, **{name: t})
            raise TypeError(f"{name} is {t.dtype}, x is {x.dtype}")
    s = x
    x, w, b = _lib.dense(x), None if w is None else _lib.dense(w), None if b is None else _lib.dense(b)
    d = None if d is None else _lib.dense(d)
    h, r = _norm(x, d, w, b, D, float(norm.eps), True)
    return h, s if d is None else r


def _embed_forward(w, ids, scale):
    out = w.new_empty(ids.shape + (w.shape[1],))
    with _lib.device_of(w):
        _lib.check(_lib.lib().lema_embedding(
            w.data_ptr(), _lib.DTYPE_CODE[w.dtype], w.shape[0], w.shape[1], ids.data_ptr(), ids.numel(),
            scale, out.data_ptr(), _lib.stream_of(w)))
    return out


def _embed_backward(ctx, gy):
    V, D, scale, padding, n = ctx.table
    ids = _lib.saved(ctx.saved_tensors[0], gy, torch.long)
    if type(gy) is not torch.Tensor or torch.is_grad_enabled() or not _unwatched(gy):
        # a graph of the backward, batched or otherwise wrapped gradients: operations that compose
        keep = (ids >= 0) & (ids < V) & (ids != padding)
        rows = torch.where(keep[..., None], gy.float() * scale, 0.0).reshape(-1, D)
        gw = torch.index_add(rows.new_zeros(V, D), 0, torch.where(keep, ids, 0).reshape(-1), rows)
        return gw.to(gy.dtype), None, None, None
    gy = _lib.dense(gy)
    gw = gy.new_empty(V, D)
    ws = gy.new_empty(n, dtype=torch.uint8)
    with _lib.device_of(gy):
        _lib.check(_lib.lib().lema_embedding_grad(
            gy.data_ptr(), _lib.DTYPE_CODE[gy.dtype], ids.data_ptr(), ids.numel(), V, D, scale, padding,
            gw.data_ptr(), ws.data_ptr(), n, _lib.stream_of(gy)))
    return gw, None, None, None


class _Embed(torch.autograd.Function):
    """The lookup, and the table's gradient by sorted tokens (its sums have a fixed order)."""

    @staticmethod
    def forward(ctx, w, ids, scale, padding):
        ctx.save_for_backward(ids)
        V, D = w.shape
        ctx.table = V, D, scale, padding, _lib.lib().lema_embedding_grad_workspace_bytes(ids.numel(), V, D)
        return _embed_forward(w, ids, scale)

    backward = staticmethod(_lib.once(_embed_backward))


class _ModelEmbed(_Embed):
    """The same in a model, whose exact op and fp32 operations have gradients of gradients."""
    backward = staticmethod(_embed_backward)


# Positions from which a model's lookup takes the gradient by sorted tokens. A lookup with its
# gradient in torch's two operations took 88 to 223 us at 2048 positions, by table (256 x 64 to
# 50,304 x 1536) and tokens (even, Zipf, all the same), and 83 to 88 so; 1024 took 51 to 123 and 82 to 94,
# 200 took 48 to 64 and 81 to 87, most of it the host's.
SORTED_GRAD_MIN = 2048

_MODULES = torch.nn.modules.module


def _plain(mod: nn.Module, kind: type = nn.Embedding) -> bool:
    """Whether a call of mod does nothing but what its kind does: an nn.Embedding (or nn.Linear)
    itself, with no hooks and no forward of its own. torch has no public names for these; one that is
    missing counts as a hook."""
    try:
        return (type(mod) is kind and "forward" not in mod.__dict__
                and not (mod._forward_hooks or mod._forward_pre_hooks or mod._backward_hooks
                         or mod._backward_pre_hooks or _MODULES._global_forward_hooks
                         or _MODULES._global_forward_pre_hooks or _MODULES._global_backward_hooks
                         or _MODULES._global_backward_pre_hooks))
    except AttributeError:
        return False


def embed(emb: nn.Embedding, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """emb(ids) * scale, rounded once, in float32, float16 or bfloat16. The ids must lie in
    [0, vocab): on the GPU one outside it gives a zero row and no gradient.

    Differentiable in the table (`padding_idx` gets a zero gradient): the gradient adds up each
    token's rows in a fixed order, in fp32. A module with hooks or with a forward of its own is
    called. So is one that renormalises its table (max_norm), wants a sparse gradient or one scaled
    by frequency, or a gradient of more than 2^20 rows, or lies on the CPU; the scale's product is
    then an operation of its own."""
    return _embed(emb, ids, scale, _Embed)


def _embed(emb, ids, scale, function):
    """embed, with the autograd Function that records it."""
    if not _plain(emb):
        y = emb(ids)
        return y if scale == 1.0 else y * scale
    w = emb.weight
    grad = _lib.needs_grad(w)
    if not (w.is_cuda and ids.device == w.device and w.dtype in _lib.DTYPE_CODE and w.is_contiguous()
            and ids.dtype in (torch.long, torch.int32) and emb.max_norm is None and w.numel()
            and w.shape[1] <= 1 << 20
            and not (grad and (emb.sparse or emb.scale_grad_by_freq or w.shape[0] > 1 << 20))):
        y = emb(ids)
        return y if scale == 1.0 else y * scale
    if ids.dtype is not torch.long or not ids.is_contiguous():
        ids = ids.long().contiguous()
    if grad:
        return function.apply(w, ids, float(scale), -1 if emb.padding_idx is None else emb.padding_idx)
    return _embed_forward(w, ids, float(scale))


def argmax_into(logits: torch.Tensor, out: torch.Tensor) -> None:
    """out[...] = logits.argmax(-1) (the first index of the maximum, NaN above every number),
    written in place: one workgroup per row of bf16 logits."""
    V = logits.shape[-1]
    if not (_fused(logits) and V % 8 == 0 and logits.data_ptr() % 16 == 0 and out.is_cuda
            and out.dtype == torch.long and out.is_contiguous()
            and out.numel() == logits.numel() // V):
        out.copy_(logits.argmax(-1).view(out.shape))
        return
    _lib.check(_lib.lib().lema_argmax_bf16(logits.data_ptr(), logits.numel() // V, V, V,
                                           out.data_ptr(), 1, _lib.stream_of(logits)))


def _swiglu_forward(g, u):
    out = torch.empty_like(g)
    _lib.check(_lib.lib().lema_swiglu_bf16(g.data_ptr(), u.data_ptr(), out.data_ptr(),
                                           g.numel(), _lib.stream_of(g)))
    return out


class _SwiGLUProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, u):
        ctx.save_for_backward(g, u)
        return _swiglu_forward(g, u)

    @staticmethod
    @_lib.once
    def backward(ctx, gy):
        gy = _lib.placed(_lib.dense(gy), 16)
        g, u = (_lib.saved(t, gy, gy.dtype, 16) for t in ctx.saved_tensors)
        gg, gu = torch.empty_like(g), torch.empty_like(u)
        with _lib.device_of(gy):
            _lib.check(_lib.lib().lema_swiglu_grad_bf16(
                g.data_ptr(), u.data_ptr(), gy.data_ptr(), gg.data_ptr(), gu.data_ptr(), g.numel(),
                _lib.stream_of(gy)))
        return gg, gu


def swiglu(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    if not (_fused(g, u) and g.shape == u.shape and g.numel() % 8 == 0):
        return F.silu(g) * u
    return _SwiGLUProduct.apply(g, u) if _lib.needs_grad(g, u) else _swiglu_forward(g, u)


def _gated_forward(x, wg, wu, keep):
    """y of gated_linear, and where asked for its derivatives by both products."""
    N, K = wg.shape
    M = x.numel() // K
    y = x.new_empty(x.shape[:-1] + (N,))
    L = _lib.lib()
    slopes = x.new_empty(L.lema_gated_linear_slopes_bytes(M, N), dtype=torch.uint8) if keep else None
    n = L.lema_gated_linear_workspace_bytes(M, N, K)
    ws = x.new_empty(n, dtype=torch.uint8) if n else None
    with _lib.device_of(x):
        _lib.check(L.lema_gated_linear(
            x.data_ptr(), wg.data_ptr(), wu.data_ptr(), _lib.DTYPE_CODE[x.dtype], M, N, K, y.data_ptr(),
            _ptr(slopes), _ptr(ws), n, _lib.stream_of(x)))
    return y, slopes


def _gated_grad_ops(gy, x, wg, wu):
    """The gradients of gated_linear in torch's operations, which have gradients of their own and compose with
    functional transforms."""
    g, u, x2 = F.linear(x, wg).float(), F.linear(x, wu).float(), x.reshape(-1, x.shape[-1])
    s = torch.sigmoid(g)
    dg, du = ((gy.float() * d).to(x.dtype) for d in (u * s * (1 + g * (1 - s)), g * s))
    gw = ((d.reshape(-1, d.shape[-1]).t() @ x2) for d in (dg, du))
    return F.linear(dg, wg.t()) + F.linear(du, wu.t()), *gw


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu):
        y, slopes = _gated_forward(x, wg, wu, True)
        ctx.save_for_backward(x, wg, wu, slopes)
        return y

    @staticmethod
    def backward(ctx, gy):
        # float16 had torch's operations before it had this kernel: what they take is taken still. (In
        # bfloat16 swiglu has no gradient of its gradient either.)
        if gy.dtype is torch.float16 and (torch.is_grad_enabled() or not _unwatched(gy)):
            grads = _gated_grad_ops(gy, *ctx.saved_tensors[:3])
            return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad))
        return _GatedLinear._kernels(ctx, gy)

    @staticmethod
    @_lib.once
    def _kernels(ctx, gy):
        gy = _lib.dense(gy)
        x, wg, wu, slopes = ctx.saved_tensors
        x, wg, wu = (_lib.saved(t, gy, gy.dtype, 16) for t in (x, wg, wu))
        slopes = _lib.saved(slopes, gy, torch.uint8, 16)
        N, K = wg.shape
        M = x.numel() // K
        want_x, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        gx = torch.empty_like(x) if want_x else None
        gwg, gwu = (torch.empty_like(wg), torch.empty_like(wu)) if want_w else (None, None)
        L = _lib.lib()
        n = L.lema_gated_linear_grad_workspace_bytes(M, N, K)
        ws = x.new_empty(n, dtype=torch.uint8)
        with _lib.device_of(gy):
            _lib.check(L.lema_gated_linear_grad(
                x.data_ptr(), wg.data_ptr(), wu.data_ptr(), slopes.data_ptr(), gy.data_ptr(),
                _lib.DTYPE_CODE[gy.dtype], M, N, K, _ptr(gx), _ptr(gwg), _ptr(gwu), ws.data_ptr(), n,
                _lib.stream_of(gy)))
        return gx, gwg, gwu


GATED_MAX_WIDTH = 1 << 20
_DENSE = (torch.Tensor, nn.Parameter)
_C, _FORWARD_AD, _compiling = torch._C, torch.autograd.forward_ad, torch.compiler.is_compiling


def _parameter(mod: nn.Module, name: str):
    """mod.name, without the module's own lookup (0.4 us) where it is a parameter."""
    ps = mod._parameters
    return ps[name] if name in ps else getattr(mod, name)


def _ordinary(x, wg, wu) -> bool:
    """Whether the tensors are nothing but memory that a kernel can be handed: no subclass, which may hold its
    numbers elsewhere, and nothing that torch traces or transforms. torch has no public names for most of
    these; one that is missing counts as a yes to them."""
    try:
        return (type(x) in _DENSE and type(wg) in _DENSE and type(wu) in _DENSE
                and not _C._are_functorch_transforms_active() and _C._len_torch_dispatch_stack() == 0
                and _FORWARD_AD._current_level < 0 and not _C._is_tracing())
    except AttributeError:
        return False


def gated_linear(x: torch.Tensor, gate: nn.Linear, up: nn.Linear) -> torch.Tensor:
    """silu(gate(x)) * up(x), the input of the feed-forward block's down projection, in one kernel on
    the GPU in bfloat16 and float16: both products in fp32, their product rounded once.
    Differentiable in x and both weights; for the gradient the forward keeps the result's derivatives by
    both products, in 20 bits. Widths that are multiples of 8, up to 2^20. Other widths, types and devices, modules
    with a bias, hooks or a forward of their own, weights of another tensor class, torch.autocast, forward mode,
    functional transforms and tracing take linear and swiglu. In float16 the gradients have gradients, in torch's
    operations."""
    if not (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16) and not _compiling()
            and _plain(gate, nn.Linear) and _plain(up, nn.Linear)):
        return swiglu(linear(x, gate), linear(x, up))
    wg, wu = _parameter(gate, "weight"), _parameter(up, "weight")
    K = x.shape[-1] if x.dim() else 0
    if not (_ordinary(x, wg, wu) and wg.dtype is wu.dtype is x.dtype
            and wg.device == wu.device == x.device and wg.shape == wu.shape and wg.dim() == 2
            and wg.shape[1] == K and K % 8 == 0 and wg.shape[0] % 8 == 0
            and 0 < K <= GATED_MAX_WIDTH and 0 < wg.shape[0] <= GATED_MAX_WIDTH
            and x.numel() and x.numel() // K < 1 << 30
            and _parameter(gate, "bias") is None and _parameter(up, "bias") is None
            and not torch.is_autocast_enabled()):
        return swiglu(linear(x, gate), linear(x, up))
    x, wg, wu = (_lib.placed(_lib.dense(t), 16) for t in (x, wg, wu))
    if _lib.needs_grad(x, wg, wu):
        return _GatedLinear.apply(x, wg, wu)
    return _gated_forward(x, wg, wu, False)[0]


class _CrossEntropySum(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, y):
        V = logits.shape[-1]
        rows = logits.numel() // V
        loss = logits.new_empty(rows, dtype=torch.float32)
        stats = logits.new_empty(rows, 2, dtype=torch.float32)
        with _lib.device_of(logits):
            _lib.check(_lib.lib().lema_cross_entropy_stats_bf16(
                logits.data_ptr(), rows, V, V, y.data_ptr(), loss.data_ptr(), stats.data_ptr(),
                _lib.stream_of(logits)))
        ctx.save_for_backward(logits, y, stats)
        return loss.sum()

    @staticmethod
    @_lib.once
    def backward(ctx, g):
        logits, y, stats = ctx.saved_tensors
        logits, y, stats = (_lib.saved(t, g, dt, align) for t, dt, align in
                            ((logits, torch.bfloat16, 1), (y, torch.long, 1), (stats, torch.float32, 8)))
        V = logits.shape[-1]
        rows = logits.numel() // V
        grad, coef = torch.empty_like(logits), -g.reshape(1)
        with _lib.device_of(g):
            _lib.check(_lib.lib().lema_token_logprobs_grad(
                logits.data_ptr(), _lib.BF16, rows, max(1, rows), V, 0, V, y.data_ptr(), None, 1.0,
                stats.data_ptr(), coef.data_ptr(), max(1, rows), None, None, 0, grad.data_ptr(),
                _lib.stream_of(g)))
        return grad, None


def cross_entropy_sum(logits: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Sum over rows of logsumexp(logits) - logits[y] (fp32), differentiable in the logits. In bf16 on
    the GPU a y outside the vocabulary makes the sum, and its row's gradient, NaN."""
    V = logits.shape[-1]
    rows = logits.numel() // V if V else 0
    if not (_fused(logits) and V and V % 8 == 0 and y.device == logits.device and y.numel() == rows):
        if V and y.shape == logits.shape[:-1]:  # the vocabulary is the last dim here, the second one there
            logits, y = logits.reshape(rows, V), y.reshape(rows)
        return F.cross_entropy(logits.float(), y, reduction="sum")
    yy = y.reshape(-1).to(torch.int64).contiguous()
    if _lib.needs_grad(logits):
        return _CrossEntropySum.apply(logits, yy)
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _lib.check(_lib.lib().lema_cross_entropy_bf16(
        logits.data_ptr(), rows, V, V, yy.data_ptr(), loss.data_ptr(), _lib.stream_of(logits)))
    return loss.sum()


SKINNY_ROWS = 32  # products with at most this many token rows run on the skinny MFMA kernel


def _skinny(x: torch.Tensor, weight: torch.Tensor) -> bool:
    K = x.shape[-1]
    return (_fused(x, weight) and K and K % 32 == 0 and weight.shape[-1] == K
            and 0 < x.numel() // K <= SKINNY_ROWS
            and x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0)


def _skinny_forward(x, w):
    K, N = x.shape[-1], w.shape[0]
    M = x.numel() // K
    y = x.new_empty(x.shape[:-1] + (N,))
    _lib.check(_lib.lib().lema_skinny_gemm_bf16(
        x.data_ptr(), K, w.data_ptr(), K, y.data_ptr(), N, M, N, K, _lib.stream_of(x)))
    return y


class _SkinnyLinear(torch.autograd.Function):
    """The skinny product where a gradient is wanted: the same y, nn.Linear's gradients."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return _skinny_forward(x, w)

    @staticmethod
    @_lib.once
    def backward(ctx, gy):
        x, w = ctx.saved_tensors
        g2 = gy.reshape(-1, gy.shape[-1])
        gx = (g2 @ w).view(x.shape) if ctx.needs_input_grad[0] else None
        gw = g2.t() @ x.reshape(-1, x.shape[-1]) if ctx.needs_input_grad[1] else None
        return gx, gw


def linear(x: torch.Tensor, lin: nn.Linear) -> torch.Tensor:
    """lin(x); a decode-shaped product (<= 32 rows, bf16) on the skinny MFMA kernel."""
    if isinstance(lin, fp8.Fp8Linear) or not _skinny(x, lin.weight):
        return lin(x)
    if _lib.needs_grad(x, lin.weight):
        return _SkinnyLinear.apply(x, lin.weight)
    return _skinny_forward(x, lin.weight)


def project_codes(x: torch.Tensor, lin: nn.Linear, d: int, code_dtype: torch.dtype):
    """[B, T, dim] -> [B, H, T] codes of lin(x) viewed as H heads of d, or None when the
    shape is not decode-sized (the caller then projects and packs)."""
    if not (_skinny(x, lin.weight) and x.dim() == 3 and _pack_tiles(d)):
        return None
    B, T, K = x.shape
    N = lin.weight.shape[0]
    codes = torch.empty((B, N // d, T), dtype=code_dtype, device=x.device)
    _lib.check(_lib.lib().lema_skinny_pack_bf16(
        x.data_ptr(), K, lin.weight.data_ptr(), K, B * T, N, K, d, T, codes.data_ptr(),
        codes.element_size(), _lib.stream_of(x)))
    return codes


def _pack_tiles(d: int) -> bool:
    """Whether the skinny kernel packs d-bit codes: heads split over 16-column blocks when d
    is a multiple of 8, else whole heads in blocks of up to 64 columns."""
    return d % 8 == 0 or any((16 * c) % d == 0 for c in (1, 2, 3, 4))


def project_qkv(x: torch.Tensor, at, code_dtype: torch.dtype, norm: nn.RMSNorm | None = None):
    """[B, T, dim] -> (qc, kc [B, H, T] codes, v [B, H, T, d_v] view) with all three
    projections in one launch (skinny MFMA kernel, pack epilogues for q and k), or None when
    the shape is not decode-sized or the heads differ in count. With `norm`, x is the layer's
    input and the launch normalises it first, rounded as rms_norm rounds it (the same codes and
    v as rms_norm followed by this, with one launch fewer); None also where that does not
    apply."""
    c = at.cfg
    wq, wk, wv = at.q_proj.weight, at.k_proj.weight, at.v_proj.weight
    if not (_skinny(x, wq) and x.dim() == 3 and _fused(wk, wv) and wq.shape == wk.shape
            and _pack_tiles(c.d_qk)):
        return None
    B, T, K = x.shape
    Nqk, Nv = wq.shape[0], wv.shape[0]
    if norm is not None:
        M = B * T
        ct = 1 if c.d_qk % 8 == 0 else next(k for k in range(1, 5) if (16 * k) % c.d_qk == 0)
        if not (_fused(norm.weight) and norm.weight.data_ptr() % 16 == 0 and x.is_contiguous()
                and K <= 2048
                and M * (K + 8) * 2 + 8 * (16 if M <= 16 else 32) * (16 * ct + 1) * 4 <= 160 * 1024):
            return None
    qc = x.new_empty((B, Nqk // c.d_qk, T), dtype=code_dtype)
    kc = torch.empty_like(qc)
    v = x.new_empty((B, T, Nv))
    if norm is not None:
        eps = norm.eps if norm.eps is not None else torch.finfo(x.dtype).eps
        _lib.check(_lib.lib().lema_skinny_norm_qkv_bf16(
            x.data_ptr(), norm.weight.data_ptr(), float(eps), wq.data_ptr(), wk.data_ptr(),
            wv.data_ptr(), K, B * T, Nqk, Nv, K, c.d_qk, T, qc.data_ptr(), kc.data_ptr(),
            qc.element_size(), v.data_ptr(), _lib.stream_of(x)))
    else:
        _lib.check(_lib.lib().lema_skinny_qkv_bf16(
            x.data_ptr(), K, wq.data_ptr(), wk.data_ptr(), wv.data_ptr(), K, B * T, Nqk, Nv, K,
            c.d_qk, T, qc.data_ptr(), kc.data_ptr(), qc.element_size(), v.data_ptr(),
            _lib.stream_of(x)))
    return qc, kc, v.view(B, T, c.num_kv_heads, c.d_v).transpose(1, 2)


# Rows of a prefill projection taken by lema_qk_pack_bf16 (q and k straight to codes): its
# 256 x 256 tiles cover the rows in 8 row groups, one per XCD.
QK_PACK_ROWS = 2048
# Whether the model's prefill takes its q and k codes from lema_qk_pack_bf16 (the codes are
# identical either way). Off: on the 4 x 16384-token, dim-1536 prefill the launch takes
# 494.5-541 us against 526-560 us for the two hipBLASLt GEMMs and two packs when timed alone,
# but 572 us against 525 us inside the forward, where both run at the clock a sustained matrix
# load holds (it spends ~30% more cycles per FLOP than the library's GEMMs); the forward's step
# time is the same with it on or off (114.5-114.8 ms).
FUSED_QK_PACK = False


def project_qk_prefill(x: torch.Tensor, at, code_dtype: torch.dtype):
    """[B, T, dim] -> (qc, kc [B, H, T] codes) of a prefill-sized input (B * T a multiple of
    2048 rows, bf16, no autograd): the query and key projections and the sign-pack in one
    persistent MFMA launch whose epilogue writes the codes, so the pre-activations zq and zk
    never reach memory. The same codes as project + pack_codes (bit j = bf16(z_j) >= 0); None
    where the launch does not apply (the caller then projects and packs)."""
    c = at.cfg
    wq, wk = at.q_proj.weight, at.k_proj.weight
    if not (_fused(x, wq, wk) and x.dim() == 3 and wq.shape == wk.shape):
        return None
    if torch.is_grad_enabled() and (x.requires_grad or wq.requires_grad or wk.requires_grad):
        return None
    B, T, K = x.shape
    N, d = wq.shape[0], c.d_qk
    cb = torch.iinfo(code_dtype).bits // 8
    if ((B * T) % QK_PACK_ROWS or N % 256 or N > 65536 or K % 64 or d % 8 or d > 64 or N % d
            or cb != (4 if d <= 32 else 8) or B * T * (N // d) * cb >= 1 << 31
            or x.data_ptr() % 16 or wq.data_ptr() % 16 or wk.data_ptr() % 16):
        return None
    qc = torch.empty((B, N // d, T), dtype=code_dtype, device=x.device)
    kc = torch.empty_like(qc)
    _lib.check(_lib.lib().lema_qk_pack_bf16(
        x.data_ptr(), K, wq.data_ptr(), wk.data_ptr(), K, B * T, N, K, d, T, qc.data_ptr(),
        kc.data_ptr(), qc.element_size(), _lib.stream_of(x)))
    return qc, kc


ATTN_KINDS = ("lema",)
POS_KINDS = ("nope",)


def _pad128(n) -> int:
    return -(-int(n) // 128) * 128


@dataclass
class ModelConfig:
    """Geometry of a LEMA model (code/lema/model.py:33-82). `d_qk`, `d_v` default to
    dim // num_heads, `dim_ff` to 8 * dim / 3; `vocab_size` and `dim_ff` are rounded up to a
    multiple of 128 (the padded vocabulary rows are never targets)."""
    vocab_size: int
    depth: int
    dim: int
    num_heads: int
    d_qk: int = 0
    d_v: int = 0
    dim_ff: int = 0
    num_kv_heads: int = 0
    attn: str = "lema"
    pos: str = "nope"
    norm_eps: float = 1e-5

    def __post_init__(self):
        if self.attn not in ATTN_KINDS:
            raise ValueError(f"attn must be one of {ATTN_KINDS} (the exact-match path), "
                             f"got {self.attn!r}")
        if self.pos not in POS_KINDS:
            raise ValueError(f"pos must be one of {POS_KINDS}, got {self.pos!r}")
        if (not self.d_qk or not self.d_v) and self.dim % self.num_heads:
            raise ValueError(f"dim {self.dim} is not divisible by num_heads {self.num_heads}")
        head = self.dim // self.num_heads
        self.d_qk = self.d_qk or head
        self.d_v = self.d_v or head
        self.dim_ff = _pad128(self.dim_ff or 8 * self.dim / 3)
        self.vocab_size = _pad128(self.vocab_size)
        self.num_kv_heads = self.num_kv_heads or self.num_heads
        if self.num_kv_heads != self.num_heads:
            raise ValueError("grouped-query attention (num_kv_heads < num_heads) is "
                             "implemented for softmax attention only")
        if self.d_qk > 64:
            raise ValueError(f"d_qk {self.d_qk} > 64: codes must pack into one uint64")

    @classmethod
    def from_dict(cls, d: dict) -> "ModelConfig":
        names = {f.name for f in dataclasses.fields(cls)}
        return cls(**{k: v for k, v in d.items() if k in names})

    def summary(self) -> str:
        return (f"{self.depth}L d{self.dim} h{self.num_heads} d_qk {self.d_qk} d_v {self.d_v} "
                f"dim_ff {self.dim_ff} attn {self.attn} pos {self.pos}")


class SwiGLU(nn.Module):
    def __init__(self, dim: int, dim_ff: int):
        super().__init__()
        self.gate = nn.Linear(dim, dim_ff, bias=False)
        self.up = nn.Linear(dim, dim_ff, bias=False)
        self.down = nn.Linear(dim_ff, dim, bias=False)

    def forward(self, x, residual=None):
        """down(silu(gate(x)) * up(x)), plus `residual` when given (Block's x + mlp(h)). On
        decode shapes the gate, up and product are one launch, rounded as gated_linear rounds
        them, and the down projection adds the residual in its epilogue; longer inputs take
        gated_linear, and in bf16 without autograd the down GEMM accumulates into `residual`
        itself, which is then returned."""
        if self._fp8():
            gated = (isinstance(self.gate, fp8.Fp8Linear) and isinstance(self.up, fp8.Fp8Linear)
                     and self.gate.out_features % 8 == 0)
            a = (fp8.gated_linear(x, self.gate.weight, self.up.weight) if gated
                 else gated_linear(x, self.gate, self.up))
            if isinstance(self.down, fp8.Fp8Linear):
                return self.down(a, residual)
            y = linear(a, self.down)
            return y if residual is None else residual + y
        g, u, dn = self.gate.weight, self.up.weight, self.down.weight
        if _skinny(x, g) and g.shape == u.shape and u.data_ptr() % 16 == 0 and u.is_contiguous() \
                and not _lib.needs_grad(x, g, u, dn, residual):
            K, N = x.shape[-1], g.shape[0]
            M = x.numel() // K
            a = x.new_empty(x.shape[:-1] + (N,))
            L = _lib.lib()
            # (widths that gated_linear does not take keep the roundings that they have there)
            _lib.check((L.lema_skinny_gated_bf16 if N % 8 == 0 else L.lema_skinny_swiglu_bf16)(
                x.data_ptr(), K, g.data_ptr(), u.data_ptr(), K, M, N, K, a.data_ptr(),
                _lib.stream_of(x)))
            if residual is not None and _skinny(a, dn) and residual.is_contiguous() \
                    and residual.shape == x.shape[:-1] + (dn.shape[0],) \
                    and residual.dtype == a.dtype and residual.data_ptr() % 16 == 0:
                y = torch.empty_like(residual)
                _lib.check(_lib.lib().lema_skinny_gemm_add_bf16(
                    a.data_ptr(), N, dn.data_ptr(), N, residual.data_ptr(), y.data_ptr(),
                    dn.shape[0], M, dn.shape[0], N, _lib.stream_of(x)))
                return y
        else:
            a = gated_linear(x, self.gate, self.up)
            if residual is not None and not _skinny(a, dn) and a.is_cuda and \
                    a.dtype == residual.dtype == dn.dtype == torch.bfloat16 and \
                    residual.is_contiguous() and not torch.is_grad_enabled():
                # the residual add in the GEMM's epilogue, accumulating into `residual` in
                # place (one rounding of x + a . W^T where the two torch ops round twice;
                # within the forward's tolerance), 2-D operands
                D = dn.shape[0]
                residual.view(-1, D).addmm_(a.reshape(-1, a.shape[-1]), dn.t())
                return residual
        y = linear(a, self.down)
        return y if residual is None else residual + y

    def _fp8(self) -> bool:
        """Whether one of the weights is held in 8 bits."""
        kind = fp8.Fp8Linear
        return isinstance(self.gate, kind) or isinstance(self.up, kind) or isinstance(self.down, kind)

    def forward_normed(self, x, d, norm: nn.RMSNorm):
        """x + d + self(norm(x + d)), Block.forward's MLP half, on decode shapes: the norm runs
        inside the gate/up launch, rounded as rms_norm rounds it, so the result equals
        `self(*reversed(rms_norm(x, norm, d)))` bit for bit with one launch fewer. None where
        that launch does not apply."""
        if self._fp8():
            return None
        g, u, dn = self.gate.weight, self.up.weight, self.down.weight
        K, N = x.shape[-1], g.shape[0]
        M = x.numel() // K
        if not (_skinny(x, g) and _fused(d, norm.weight) and d.shape == x.shape
                and g.shape == u.shape and _fused(u) and u.data_ptr() % 16 == 0
                and d.data_ptr() % 16 == 0 and norm.weight.data_ptr() % 16 == 0 and K <= 2048
                and M * (K + 8) * 2 + 8 * (16 if M <= 16 else 32) * 33 * 4 <= 160 * 1024
                and _fused(dn) and dn.data_ptr() % 16 == 0 and N % 32 == 0):
            return None
        xo = torch.empty_like(x)
        a = x.new_empty(x.shape[:-1] + (N,))
        eps = norm.eps if norm.eps is not None else torch.finfo(x.dtype).eps
        _lib.check(_lib.lib().lema_skinny_norm_gated_bf16(
            x.data_ptr(), d.data_ptr(), norm.weight.data_ptr(), float(eps), xo.data_ptr(),
            g.data_ptr(), u.data_ptr(), K, M, N, K, a.data_ptr(), _lib.stream_of(x)))
        y = torch.empty_like(xo)
        _lib.check(_lib.lib().lema_skinny_gemm_add_bf16(
            a.data_ptr(), N, dn.data_ptr(), N, xo.data_ptr(), y.data_ptr(), dn.shape[0], M,
            dn.shape[0], N, _lib.stream_of(x)))
        return y


class Attention(nn.Module):
    """A LEMA attention block (code/lema/model.py:143-210): q, k, v projections viewed as
    `[B, H, T, d]` (transposed views, read in place by the kernels), the exact op, o_proj."""

    def __init__(self, cfg: ModelConfig):
        super().__init__()
        self.cfg = cfg
        self.kind = cfg.attn
        self.q_proj = nn.Linear(cfg.dim, cfg.num_heads * cfg.d_qk, bias=False)
        self.k_proj = nn.Linear(cfg.dim, cfg.num_kv_heads * cfg.d_qk, bias=False)
        self.v_proj = nn.Linear(cfg.dim, cfg.num_kv_heads * cfg.d_v, bias=False)
        self.o_proj = nn.Linear(cfg.num_heads * cfg.d_v, cfg.dim, bias=False)
        self.hard = False

    def project(self, x):
        """`[B, T, dim]` -> query and key pre-activations and values, `[B, H, T, d]`."""
        B, T, _ = x.shape
        c = self.cfg
        zq = linear(x, self.q_proj).view(B, T, c.num_heads, c.d_qk).transpose(1, 2)
        zk = linear(x, self.k_proj).view(B, T, c.num_kv_heads, c.d_qk).transpose(1, 2)
        v = linear(x, self.v_proj).view(B, T, c.num_kv_heads, c.d_v).transpose(1, 2)
        return zq, zk, v

    def merge(self, y):
        B, _, T, _ = y.shape
        return linear(y.transpose(1, 2).reshape(B, T, -1).contiguous(), self.o_proj)

    def forward(self, x):
        if not self.hard:
            raise NotImplementedError("only the exact (hard) op is implemented: call "
                                      "model.set_hard(True)")
        codes = (project_qk_prefill(x, self, code_dtype_for(self.cfg.d_qk))
                 if FUSED_QK_PACK else None)
        if codes is not None:  # q and k straight to codes; v by its own product
            B, T, _ = x.shape
            c = self.cfg
            v = linear(x, self.v_proj).view(B, T, c.num_kv_heads, c.d_v).transpose(1, 2)
            return self.merge(lema_from_codes(codes[0], codes[1], v))
        zq, zk, v = self.project(x)
        return self.merge(lema_hard(zq, zk, v))


def _cached(x: torch.Tensor):
    """What a forward with a cache runs in: the exchange has no gradient, and neither do the fused
    bf16 launches around it."""
    return torch.no_grad() if x.is_cuda and x.dtype is torch.bfloat16 else contextlib.nullcontext()


class Block(nn.Module):
    def __init__(self, cfg: ModelConfig):
        super().__init__()
        self.norm1 = nn.RMSNorm(cfg.dim, eps=cfg.norm_eps)
        self.attn = Attention(cfg)
        self.norm2 = nn.RMSNorm(cfg.dim, eps=cfg.norm_eps)
        self.mlp = SwiGLU(cfg.dim, cfg.dim_ff)
        self.seg = None

    def pre_attn(self, x):
        """The attention's input norm1(x): in bf16 on the device the fused norm kernel, which
        rounds x * rsqrt(mean(x^2) + eps) * w once from fp32 as torch's RMSNorm does (the
        codes are the signs of its projections)."""
        return rms_norm(x, self.norm1)[0]

    def gpu_pre(self, x):
        """Normalise, project, pack both codes (code/lema/model.py:224-227). On decode shapes
        the norm and the three projections are one launch, q and k going straight to codes
        (skinny MFMA kernel: pre-norm prologue, pack epilogues); with FUSED_QK_PACK set, on
        prefill chunks of 2048 or more rows q and k go straight to codes in one persistent
        MFMA launch."""
        at, c = self.attn, self.attn.cfg
        ct = code_dtype_for(c.d_qk)
        fused = project_qkv(x, at, ct, norm=self.norm1)
        if fused is not None:
            return fused
        h = self.pre_attn(x)
        fused = project_qkv(h, at, ct)
        if fused is not None:
            return fused
        codes = project_qk_prefill(h, at, ct) if FUSED_QK_PACK else None
        if codes is not None:  # prefill chunks of 2048+ rows
            B, T, _ = h.shape
            v = linear(h, at.v_proj).view(B, T, c.num_kv_heads, c.d_v).transpose(1, 2)
            return codes[0], codes[1], v
        qc = project_codes(h, at.q_proj, c.d_qk, ct)
        kc = project_codes(h, at.k_proj, c.d_qk, ct) if qc is not None else None
        if kc is not None:
            B, T, _ = h.shape
            v = linear(h, at.v_proj).view(B, T, c.num_kv_heads, c.d_v).transpose(1, 2)
            return qc, kc, v
        zq, zk, v = at.project(h)
        return pack_codes(zq, ct), pack_codes(zk, ct), v

    def gpu_post(self, x, got):
        """Merge the retrieved values and finish the layer (code/lema/model.py:229-232); on
        decode shapes the MLP's pre-norm runs inside its gate/up launch."""
        d = self.attn.merge(got)
        y = self.mlp.forward_normed(x, d, self.norm2)
        if y is not None:
            return y
        h, x = rms_norm(x, self.norm2, d)
        return self.mlp(h, residual=x)

    def forward(self, x, store=None):
        if store is not None:
            pre, post = self.seg or (self.gpu_pre, self.gpu_post)
            with _cached(x):
                qc, kc, v = pre(x)
                return post(x, store.exchange(qc, kc, v))
        h, x = rms_norm(x, self.norm2, self.attn(self.pre_attn(x)))
        return self.mlp(h, residual=x)


class Transformer(nn.Module):
    def __init__(self, cfg: ModelConfig):
        super().__init__()
        self.cfg = cfg
        self.tok_emb = nn.Embedding(cfg.vocab_size, cfg.dim)
        self.blocks = nn.ModuleList(Block(cfg) for _ in range(cfg.depth))
        self.norm_f = nn.RMSNorm(cfg.dim, eps=cfg.norm_eps)
        self.lm_head = nn.Linear(cfg.dim, cfg.vocab_size, bias=False)
        self.checkpoint_blocks = False
        self._init_weights()

    def _init_weights(self):
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.normal_(m.weight, mean=0.0, std=1.0 / math.sqrt(m.weight.shape[1]))
            elif isinstance(m, nn.Embedding):
                nn.init.normal_(m.weight, mean=0.0, std=1.0 / math.sqrt(self.cfg.dim))
        for b in self.blocks:
            for lin in (b.attn.o_proj, b.mlp.down):
                lin.weight.data.mul_(1.0 / math.sqrt(2 * self.cfg.depth))

    def lema_layers(self):
        return [b.attn for b in self.blocks if b.attn.kind == "lema"]

    def set_hard(self, hard: bool = True):
        for att in self.lema_layers():
            att.hard = hard

    def new_cache(self, place: str = "hbm", **kw):
        """A retrieval cache for this model (code/lema/model.py:306-324): in device memory
        (place "hbm", or "vram"), or in pinned host RAM ("ram", the reference's placement,
        for caches larger than device memory; the same kernels work on it in place over the
        host link). `max_cache_len=` or `capacity=` slots, `batch=`, `max_load=`,
        `codes_hook=` as in `LemaCache`."""
        from .cache import LemaCache
        if place not in ("hbm", "vram", "ram"):
            raise ValueError(f"a LEMA cache lives in device memory (place='hbm') or host RAM "
                             f"(place='ram'); place={place!r} is not an implementation of it")
        p = next(self.parameters())
        kw.setdefault("dtype", p.dtype)
        kw.pop("pin", None)
        return LemaCache(self.cfg, device=p.device, place="ram" if place == "ram" else "hbm",
                         **kw)

    def forward(self, idx, *, cache=None, return_logits=True):
        """Run `idx` through the model (code/lema/model.py:337-363).

            forward(x)                                batched, no state
            forward(x, cache=c, return_logits=False)  prefill: fills c, no logits
            forward(next, cache=c)                    extending c

        With a cache, queries match keys from before this call too, so a sequence can be fed
        in pieces; any chunking gives the one-shot result but for last bits, which can depend on
        how many rows a call has: fp32 sums take another order, and in bf16 on the GPU a block of
        more than 32 rows adds its residual before the down product is rounded, one of fewer
        after. There nothing of a call with a cache has a gradient, its logits neither. Tokens must lie in [0, vocab_size); on the
        GPU they are not checked.
        """
        if cache is not None and not (self.lema_layers()
                                      and all(a.hard for a in self.lema_layers())):
            raise ValueError("a cache needs an all-LEMA model in hard mode")
        x = self._embed(idx) if cache is None else self.tok_emb(idx)
        with _cached(x) if cache is not None else contextlib.nullcontext():
            for li, blk in enumerate(self.blocks):
                x = blk(x, store=(cache.layer(li) if cache is not None else None))
            if cache is not None:
                cache.t += idx.shape[-1]
            return linear(rms_norm(x, self.norm_f)[0], self.lm_head) if return_logits else None

    def _embed(self, idx):
        """The token rows: `embed`, whose gradient sorts the tokens, where one of many is wanted."""
        emb = self.tok_emb
        if idx.numel() >= SORTED_GRAD_MIN and _plain(emb) and _lib.needs_grad(emb.weight):
            return _embed(emb, idx, 1.0, _ModelEmbed)
        return emb(idx)

    def hidden(self, idx):
        """The final normalised hidden states (the input of lm_head), without a cache."""
        x = self._embed(idx)
        for blk in self.blocks:
            x = blk(x)
        return rms_norm(x, self.norm_f)[0]

    def n_params(self, embedding: bool = True) -> int:
        n = sum(p.numel() for p in self.parameters())
        n += sum(m.out_features * m.in_features for m in self.modules() if isinstance(m, fp8.Fp8Linear))
        if not embedding:
            n -= self.tok_emb.weight.numel() + self.lm_head.out_features * self.lm_head.in_features
        return n


def lm_loss(model: Transformer, x: torch.Tensor, y: torch.Tensor, chunk: int = 4096):
    """Mean next-token cross-entropy without holding the full `[B, T, vocab]` logits: the
    head and the loss run `chunk` positions at a time on the final hidden states, in fp32
    (code/lema/train.py:131-152). Differentiable; a backward keeps the chunks' logits until then.
    At B4 T16384 with a 50,304-word vocabulary, chunks of 4096 positions (head GEMMs of 16,384
    rows, 1.65 GB of bf16 logits at a time) took the whole forward from 119.9-120.4 to
    118.2-118.8 ms against chunks of 1024."""
    h = model.hidden(x)
    total = torch.zeros((), dtype=torch.float32, device=h.device)
    for a in range(0, x.shape[1], chunk):
        # a contiguous 2-D block: the head is then one plain GEMM (a strided 3-D slice would
        # make matmul broadcast the transposed weight into a batched product instead)
        hc = h[:, a:a + chunk].reshape(-1, h.shape[-1]).contiguous()
        total += cross_entropy_sum(model.lm_head(hc), y[:, a:a + chunk].reshape(-1))
    return total / y.numel()


def load_trained(path, device="cuda") -> tuple[Transformer, ModelConfig]:
    """A finished training run, ready to evaluate (code/lema/model.py:420-436): `path` is the
    run directory (its `model.pt`) or a checkpoint file, a dict holding `config` (the
    ModelConfig fields) and `state_dict`. The model comes back in hard mode, fp32, in eval
    mode; parameters the checkpoint holds beyond this model's are dropped. Linear layers that
    it holds in 8 bits (`fp8.quantize_feed_forward`) come back so.

    The file is read with `torch.load(weights_only=True)`, which builds tensors and plain
    containers only and executes nothing from the file; a checkpoint that needs arbitrary
    objects to load raises instead. Only all-LEMA configurations load (ModelConfig raises
    ValueError for the others)."""
    path = Path(path)
    if path.is_dir():
        path = path / "model.pt"
    ck = torch.load(path, map_location="cpu", weights_only=True)
    if not isinstance(ck, dict) or "config" not in ck or "state_dict" not in ck:
        raise ValueError(f"{path}: expected a dict with 'config' and 'state_dict'")
    cfg = ModelConfig.from_dict(dict(ck["config"]))
    model = Transformer(cfg).to(device).eval()
    for name, mod in list(model.named_modules()):
        if isinstance(mod, nn.Linear) and name + ".scales" in ck["state_dict"]:
            owner, _, leaf = name.rpartition(".")
            setattr(model.get_submodule(owner), leaf,
                    fp8.Fp8Linear.blank(mod.out_features, mod.in_features, device))
    keep = model.state_dict().keys()
    model.load_state_dict({k: v for k, v in ck["state_dict"].items() if k in keep})
    model.set_hard(True)
    return model, cfg
