"""Products in 8-bit floating point for serving: half of bf16's weight bytes, and the matrix cores' 8-bit
rate in a prefill.

    quantize(x, block_rows)          e4m3 values with a power-of-two scale for each block of 128
    matmul(a, w)                     a . w^T of quantized operands
    linear(x, w)                     the same with x quantized on the way
    gated_linear(x, gate, up)        silu(x . gate^T) * (x . up^T)
    Fp8Linear, quantize_feed_forward a model's projections held so

A block is 128 columns of one row (activations) or of 128 rows (weights). Its scale is the least power
of two 2^e, e >= -126, that brings its largest finite value to at most 448, so that x / 2^e is exact and
a value is rounded once, to the nearest e4m3, halves to even; the scales are held as e8m0. A block of
zeros has the scale 1. Infinities and NaN become NaN, and reach their row (or weight's column) of the
result. Products are summed up in fp32. Into bfloat16 and float16 those of 8 consecutive columns go by an
instruction that aligns them to the largest of them and cuts off what lies 2^-13 below it (1.4e-5 of the
products' norm on random blocks). Into float32 every product is exact, at half of the speed, and the
values are those that bfloat16 holds: infinite from 2^128 on, in steps of 2^-133 below 2^-126. Nothing
here has a gradient.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

from . import _lib

__all__ = ["Fp8", "quantize", "dequantize", "matmul", "linear", "gated_linear", "Fp8Linear",
           "quantize_feed_forward"]

BLOCK = 128
MAX_WIDTH = 1 << 20
SMALL_ROWS = 32  # rows that the launch for decode steps takes, quantizing them itself


class Fp8(NamedTuple):
    """[..., columns] in 8 bits: values [..., Kp] in float8_e4m3fn, Kp the columns in whole blocks
    with zeros behind the last one, and scales in float8_e8m0fnu: [..., Kp / 128] with one for each
    row, or [rows / 128 rounded up, Kp / 128] of a matrix with one for 128 rows."""
    values: torch.Tensor
    scales: torch.Tensor
    columns: int


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _no_grad(*ts):
    if _lib.needs_grad(*ts):
        raise RuntimeError("8-bit products have no gradient: call them under torch.no_grad()")


def _quantize(x, M, K, block_rows):
    """(values [M, Kp], scales) of M rows of K; the scales as the kernels read them."""
    kb = _blocks(K)
    values = x.new_empty((M, kb * BLOCK), dtype=torch.float8_e4m3fn)
    shape = (kb, -(-M // 4) * 4) if block_rows == 1 else (_blocks(M), kb)
    scales = x.new_empty(shape, dtype=torch.float8_e8m0fnu)
    with _lib.device_of(x):
        _lib.check(_lib.lib().lema_fp8_quantize(
            x.data_ptr(), _lib.DTYPE_CODE[x.dtype], M, K, K, block_rows, values.data_ptr(),
            scales.data_ptr(), shape[1], _lib.stream_of(x)))
    return values, scales


def quantize(x: torch.Tensor, block_rows: int = 1) -> Fp8:
    """x [..., K] in blocks of 128 columns of each row, or (block_rows=128) a matrix [N, K] in blocks of
    128 x 128. float32, float16 or bfloat16 on the device."""
    _lib.require_device(x)
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"quantize takes float32, float16 or bfloat16, got {x.dtype}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} columns are quantized, got {tuple(x.shape)}")
    if block_rows == BLOCK and x.dim() != 2:
        raise ValueError(f"blocks of {BLOCK} rows are a matrix's, got {tuple(x.shape)}")
    _no_grad(x)
    x = _lib.dense(x)
    K, lead = x.shape[-1], x.shape[:-1]
    M = x.numel() // K
    values, scales = _quantize(x, M, K, block_rows)
    if block_rows == 1:
        scales = scales[:, :M].t().view(lead + (_blocks(K),))
        values = values.view(lead + (-1,)) if M else values.new_empty(lead + (_blocks(K) * BLOCK,))
    return Fp8(values, scales, K)


def dequantize(a: Fp8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The numbers that a stands for, [..., columns], rounded to dtype."""
    rows = a.values.reshape(-1, a.values.shape[-1])
    kb = rows.shape[1] // BLOCK
    s = a.scales.float()
    if a.scales.shape[:-1] != a.values.shape[:-1]:
        s = s.repeat_interleave(BLOCK, 0)[:rows.shape[0]]
    x = rows.float().view(-1, kb, BLOCK) * s.reshape(-1, kb, 1)
    return x.view(a.values.shape)[..., :a.columns].to(dtype)


def _weight(name: str, w: Fp8, K: int, like: torch.Tensor):
    """(values, scales) of an [N, K] weight as the kernels read them."""
    v, s = w.values, w.scales
    if v.dtype is not torch.float8_e4m3fn or s.dtype is not torch.float8_e8m0fnu:
        raise TypeError(f"{name} must hold float8_e4m3fn values and float8_e8m0fnu scales, got {v.dtype} and {s.dtype}")
    if w.columns != K:
        raise ValueError(f"{name} has {w.columns} columns, the input {K}")
    kb = _blocks(K)
    if v.dim() != 2 or v.shape[1] != kb * BLOCK or not 1 <= v.shape[0] <= MAX_WIDTH:
        raise ValueError(f"{name}'s values {tuple(v.shape)} are not [N, {kb * BLOCK}], N at most {MAX_WIDTH}")
    if s.shape != (_blocks(v.shape[0]), kb):
        raise ValueError(f"{name}'s scales {tuple(s.shape)} are not [{_blocks(v.shape[0])}, {kb}]")
    if v.device != like.device or s.device != like.device:
        _lib.same_device(like, **{name: v, f"{name}'s scales": s})
    if not v.is_contiguous() or v.data_ptr() % 16:
        v = _lib.placed(v.contiguous(), 16)
    return v, s if s.is_contiguous() else s.contiguous()


def _result_type(dtype):
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"8-bit products take and give float32, bfloat16 or float16, not {dtype}")


def _product(values, scales, lds, M, K, w, w2, dtype, shape):
    """values [M, Kp] with block-major scales times one weight, or gated by a second one."""
    (v, s), (v2, s2) = w, w2 or (None, None)
    N = v.shape[0]
    out = values.new_empty(shape + (N,), dtype=dtype)
    L = _lib.lib()
    wide = dtype is torch.float32
    size = L.lema_fp8_matmul_f32_workspace_bytes if wide else L.lema_fp8_matmul_workspace_bytes
    n = size(M, N, K, w2 is not None)
    ws = values.new_empty(n, dtype=torch.uint8) if n else None
    operands = (values.data_ptr(), scales.data_ptr(), lds, v.data_ptr(), s.data_ptr(), _ptr(v2), _ptr(s2))
    rest = (M, N, K, out.data_ptr(), _ptr(ws), n, _lib.stream_of(values))
    with _lib.device_of(values):
        _lib.check(L.lema_fp8_matmul_f32(*operands, *rest) if wide else
                   L.lema_fp8_matmul(*operands, _lib.DTYPE_CODE[dtype], *rest))
    return out


def matmul(a: Fp8, w: Fp8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a . w^T: a [..., K] with a scale for each row's blocks, w [N, K] with one for each 128 x 128;
    [..., N] in float32, bfloat16 or float16."""
    _result_type(dtype)
    K, lead = a.columns, a.values.shape[:-1]
    _lib.require_device(a.values, a.scales)
    kb = _blocks(K)
    if a.values.dtype is not torch.float8_e4m3fn or a.scales.dtype is not torch.float8_e8m0fnu:
        raise TypeError(f"a must hold float8_e4m3fn values and float8_e8m0fnu scales, got {a.values.dtype} "
                        f"and {a.scales.dtype}")
    if not 1 <= K <= MAX_WIDTH or a.values.shape[-1:] != (kb * BLOCK,) or a.scales.shape != lead + (kb,):
        raise ValueError(f"a's values {tuple(a.values.shape)} and scales {tuple(a.scales.shape)} are not those of "
                         f"rows of {K} columns with a scale for each of {kb} blocks")
    _lib.same_device(a.values, **{"a's scales": a.scales})
    w = _weight("w", w, K, a.values)
    values = _lib.placed(a.values.contiguous(), 16)
    M = values.numel() // (kb * BLOCK)
    if M == 0:
        return values.new_empty(lead + (w[0].shape[0],), dtype=dtype)
    scales = a.scales.reshape(M, kb)
    lds = scales.stride(1)
    if scales.stride(0) != 1 or lds % 4 or lds < M or scales.data_ptr() % 4 \
            or scales.storage_offset() + kb * lds > scales.untyped_storage().nbytes():
        lds = -(-M // 4) * 4
        s = scales.new_empty((kb, lds))
        s[:, :M].copy_(scales.t())
        scales = s
    return _product(values, scales, lds, M, K, w, None, dtype, lead)


def _linear(x, w, w2, residual):
    """x [..., K] through one weight (plus a residual), or through a gate and a second one."""
    K = x.shape[-1]
    lead = x.shape[:-1]
    x = _lib.dense(x)
    M = x.numel() // K
    N = w[0].shape[0]
    if M == 0:
        return x.new_empty(lead + (N,))
    if M > SMALL_ROWS:
        values, scales = _quantize(x, M, K, 1)
        y = _product(values, scales, scales.shape[1], M, K, w, w2, x.dtype, lead)
        return y if residual is None else y.add_(residual)
    out = x.new_empty(lead + (N,))
    (v, s), (v2, s2) = w, w2 or (None, None)
    L = _lib.lib()
    rest = (K, v.data_ptr(), s.data_ptr(), _ptr(v2), _ptr(s2), _ptr(residual), M, N, K, out.data_ptr(), _lib.stream_of(x))
    with _lib.device_of(x):
        _lib.check(L.lema_fp8_linear_f32(x.data_ptr(), *rest) if x.dtype is torch.float32 else
                   L.lema_fp8_linear(x.data_ptr(), _lib.DTYPE_CODE[x.dtype], *rest))
    return out


def _input(x, *others):
    _lib.require_device(x)
    _result_type(x.dtype)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rows of 1 to {MAX_WIDTH} columns are taken, got {tuple(x.shape)}")
    _no_grad(x, *others)


def linear(x: torch.Tensor, w: Fp8, residual: torch.Tensor | None = None) -> torch.Tensor:
    """x . w^T (+ residual) in x's type, x [..., K] in float32, bfloat16 or float16, quantized for each
    row's blocks: one launch up to 32 rows, a quantizing pass and a product beyond. The product is rounded
    to x's type before the residual [..., N] is added."""
    _input(x, residual)
    w = _weight("w", w, x.shape[-1], x)
    if residual is not None:
        if residual.shape != x.shape[:-1] + (w[0].shape[0],):
            raise ValueError(f"the residual {tuple(residual.shape)} does not match the result "
                             f"{tuple(x.shape[:-1]) + (w[0].shape[0],)}")
        if residual.dtype is not x.dtype:
            raise TypeError(f"the residual is {residual.dtype}, x is {x.dtype}")
        _lib.same_device(x, residual=residual)
        residual = _lib.dense(residual)
    return _linear(x, w, None, residual)


def gated_linear(x: torch.Tensor, gate: Fp8, up: Fp8) -> torch.Tensor:
    """silu(x . gate^T) * (x . up^T), x quantized once, both products in fp32, rounded once; [N, K]
    weights with N a multiple of 8."""
    _input(x)
    K = x.shape[-1]
    g, u = _weight("gate", gate, K, x), _weight("up", up, K, x)
    if g[0].shape != u[0].shape:
        raise ValueError(f"gate has {g[0].shape[0]} outputs, up {u[0].shape[0]}")
    if g[0].shape[0] % 8:
        raise ValueError(f"{g[0].shape[0]} outputs: a gated product takes a multiple of 8")
    return _linear(x, g, u, None)


class Fp8Linear(nn.Module):
    """A linear layer without bias whose weight is held in 8 bits, for inference. The bytes are buffers
    (a module's `.to(dtype)` leaves them as they are)."""

    def __init__(self, weight: Fp8):
        super().__init__()
        self.out_features, self.in_features = weight.values.shape[0], weight.columns
        self.register_buffer("values", weight.values.view(torch.uint8))
        self.register_buffer("scales", weight.scales.view(torch.uint8))

    @classmethod
    def of(cls, lin: nn.Linear) -> "Fp8Linear":
        """lin's weight, quantized in blocks of 128 x 128."""
        if lin.bias is not None:
            raise ValueError("an 8-bit linear layer has no bias")
        return cls(quantize(lin.weight.detach(), BLOCK))

    @classmethod
    def blank(cls, out_features: int, in_features: int, device=None) -> "Fp8Linear":
        """A weight of zeros, to load a state_dict into."""
        kb = _blocks(in_features)
        values = torch.zeros(out_features, kb * BLOCK, dtype=torch.uint8, device=device)
        scales = torch.full((_blocks(out_features), kb), 127, dtype=torch.uint8, device=device)
        return cls(Fp8(values.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), in_features))

    @property
    def weight(self) -> Fp8:
        return Fp8(self.values.view(torch.float8_e4m3fn), self.scales.view(torch.float8_e8m0fnu), self.in_features)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        return linear(x, self.weight, residual)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"


def quantize_feed_forward(model: nn.Module, head: bool = False) -> nn.Module:
    """Holds the feed-forward weights of a Transformer's blocks (and with `head` the head's) in 8 bits, in
    place, for serving; returns the model. The query and key projections keep their type: their
    outputs' signs are the codes that are matched exactly, and the value and output projections are
    small beside the feed-forward ones. A model's state_dict then loads into one that was held so, too.

    It pays in prefills (3 to 20% in a bf16 model of 24 layers of 1536) and in decode steps of 16 streams
    (1%) and more (32: 10%); steps of one to four streams take 18 to 25% longer."""
    for block in model.blocks:
        for name in ("gate", "up", "down"):
            lin = getattr(block.mlp, name)
            if not isinstance(lin, Fp8Linear):
                setattr(block.mlp, name, Fp8Linear.of(lin))
    if head and not isinstance(model.lm_head, Fp8Linear):
        model.lm_head = Fp8Linear.of(model.lm_head)
    return model
