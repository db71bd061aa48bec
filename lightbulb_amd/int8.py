"""Linears in 8-bit integers with a scale for each token and channel, and the norms between them.

A weight is int8 codes [n, k] and one f32 scale a channel, as W8A8 checkpoints have them; an input's
tokens are quantised to int8 as they come, one f32 scale a token, and the sums of code products are
exact:

* ``quantize_tokens``     values to codes and scales
* ``Int8Linear``          the product with one weight; ``int8_linear_group`` with up to four that read
                          one input (q, k and v), ``int8_gate_up_silu`` ``silu(gate) * up`` of a pair
* ``residual_norm``       the residual stream's update by a block's output and the norm in front of
                          the next block, as values or straight as the next products' codes

They stand beside ``quantized.QMatMul``: ``QuantizableLinear.from_int8`` puts an ``Int8Linear`` into
``quantized.Mlp``, ``attention.Attention`` and ``block.Block``, the projections of the reference's blocks
(src/model/custom_transformer_block.rs, mlp_wrapper.rs:190-195, custom_attention.rs:265-267, :671).
The arithmetic runs in liblbq's HIP kernels; torch provides memory and the current stream.
"""
from __future__ import annotations

import ctypes
import struct
from operator import attrgetter

import torch

from . import _lib
from .quantized import GROUP_MAX, _ctxs, _stream, context

#: element types of values -> the library's type ids
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
#: addresses as the library takes a list of them
_ADDRESSES = [struct.Struct(f"={n}Q").pack for n in range(GROUP_MAX + 1)]
_KINDS = {"rms": 0, "layer": 1}
MAX_K = 131071  # sums of 2^14 k stay below 2^31
NORM_MAX_K = 32768
_FUSED_ROWS, _FUSED_CODES, _FUSED_CHANNELS = 4, 16384, 16384  # LBQ_I8_FUSED_ROWS, .._CODES, .._CHANNELS


def _row(k: int) -> int:
    """LBQ_I8_ROW: the bytes of a row of k codes."""
    return (k + 127) // 128 * 128


def _values(name: str, xs: torch.Tensor) -> tuple[int, int, int]:
    """(type id, rows, elements between rows) of values [.., k] with contiguous rows evenly apart."""
    t = _DTYPES.get(xs.dtype)
    if t is None:
        raise ValueError(f"{name} must be f32, f16 or bf16, got {xs.dtype}")
    shape = xs.shape
    if len(shape) < 2:
        raise ValueError(f"{name} has only one dimension {tuple(shape)}")
    k = shape[-1]
    if xs.is_contiguous():
        return t, shape[0] if len(shape) == 2 else xs.numel() // max(k, 1), k
    strides = xs.stride()
    m, stride, step = 1, 0, None
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n != 1:
            if step is not None and s != step:
                raise ValueError(f"{name} {tuple(shape)} of strides {strides}: rows must be evenly apart")
            stride = s if step is None else stride
            step = s * n
        m *= n
    if k > 1 and strides[-1] != 1:
        raise ValueError(f"{name} {tuple(shape)} of strides {strides}: rows must be contiguous")
    return t, m, stride


def _context(dev: torch.device) -> int:
    return _ctxs.get(dev.index) or context(dev)


def _vector(name: str, t: torch.Tensor, n: int, device) -> None:
    if t.dtype != torch.float32 or t.dim() != 1 or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{name} must be a contiguous f32 tensor of {n} values, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} on {t.device}, expected {device}")


class _Fixed:
    """What the library is given as addresses when the object is made: setting such an attribute anew would
    leave the library with the old ones.  The tensors' contents may change."""

    def __setattr__(self, name, value):
        raise AttributeError(f"a {type(self).__name__}'s {name} is fixed when it is made")


# ---------------------------------------------------------------------------
# codes
# ---------------------------------------------------------------------------
class Int8Tokens:
    """Tokens as ``codes`` int8 [.., k] and ``scales`` f32 [..]: a value is code * scale.  Made by
    ``quantize_tokens`` and ``residual_norm``; ``dtype`` is that of the values they stand for."""

    # (what the products take by address goes together: the attributes cannot be set, the tensors' contents may change)
    __slots__ = ("_rows", "_scales", "_shape", "_dtype", "_device")
    scales, shape, dtype, device = (property(attrgetter(name)) for name in __slots__[1:])

    def __init__(self, rows: torch.Tensor, scales: torch.Tensor, shape: torch.Size, dtype: torch.dtype, device: torch.device):
        self._rows, self._scales, self._shape, self._dtype, self._device = rows, scales, shape, dtype, device

    @property
    def codes(self) -> torch.Tensor:
        rows, shape = self._rows, self._shape
        if rows.shape == shape:
            return rows
        rows = rows.narrow(1, 0, shape[-1])
        return rows if len(shape) == 2 else rows.unflatten(0, shape[:-1])

    def dequantize(self) -> torch.Tensor:
        """The values that the codes stand for, f32."""
        return self.codes.float() * self.scales[..., None]

    def __repr__(self) -> str:
        return f"Int8Tokens(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def _empty_tokens(shape, m: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    # (sizes one by one: 1.3 us each where a tuple of them takes 1.7)
    return (torch.empty(m, (shape[-1] + 127) // 128 * 128, dtype=torch.int8, device=device),
            torch.empty(*shape[:-1], dtype=torch.float32, device=device))


def quantize_tokens(xs: torch.Tensor) -> Int8Tokens:
    """Each row of ``xs`` [.., k] as int8 codes and one scale, its largest magnitude / 127; codes are the nearest,
    ties to even.  A row with a value that is not finite has the scale NaN and codes 0."""
    t, m, stride = _values("xs", xs)
    shape, dev = xs.shape, xs.device
    rows, scales = _empty_tokens(shape, m, dev)
    _lib.check(_lib.lib().lbq_i8_quantize(_context(dev), t, xs.data_ptr(), stride, m, shape[-1], rows.data_ptr(), scales.data_ptr(), _stream(dev)))
    return Int8Tokens(rows, scales, shape, xs.dtype, dev)


class Int8Weight(_Fixed):
    """A weight's ``codes`` int8 [n, k] and ``scales`` f32 [n], one a channel.  Rows are held 128 bytes or a multiple
    apart: codes whose k is not such are copied once, others are used as they are."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.int8 or codes.dim() != 2 or not all(codes.shape):
            raise ValueError(f"codes must be an int8 tensor [n, k], got {codes.dtype} {tuple(codes.shape)}")
        n, k = codes.shape
        if k > MAX_K:
            raise ValueError(f"k = {k} exceeds {MAX_K}")
        _vector("scales", scales, n, codes.device)
        if k % 128 or not codes.is_contiguous() or codes.data_ptr() % 16:
            rows = torch.zeros(n, _row(k), dtype=torch.int8, device=codes.device)
            rows[:, :k] = codes
        else:
            rows = codes
        self._init(rows, scales, k)

    def _init(self, rows, scales, k):
        vars(self).update(_rows=rows, codes=rows[:, :k], scales=scales, device=rows.device)

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Int8Weight":
        """f32, f16 or bf16 values [n, k]: a channel's scale is its largest magnitude / 127."""
        if w.dim() != 2 or not all(w.shape):
            raise ValueError(f"Int8Weight.quantize expects a 2-D (n, k) tensor, got {tuple(w.shape)}")
        t = quantize_tokens(w)
        self = cls.__new__(cls)
        self._init(t._rows, t.scales, w.shape[1])
        return self

    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)

    def dequantize(self) -> torch.Tensor:
        return self.codes.float() * self.scales[:, None]

    def __repr__(self) -> str:
        return f"Int8Weight(shape={self.shape()}, device={self.device})"


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
class Int8Linear(_Fixed):
    """``x W^T + bias`` over an ``Int8Weight``; bias f32 [n] or None."""

    def __init__(self, weight: Int8Weight, bias: torch.Tensor | None = None):
        n, k = weight.shape()
        if bias is not None:
            _vector("bias", bias, n, weight.device)
        arg = _lib.I8WeightStruct(weight._rows.data_ptr(), weight.scales.data_ptr(), bias.data_ptr() if bias is not None else None, n)
        at = ctypes.addressof(arg)
        vars(self).update(weight=weight, bias=bias, device=weight.device, _n=n, _k=k, _arg=arg, _at=at, _list=_ADDRESSES[1](at),
                          _ctx=context(weight.device))

    def forward(self, xs: "torch.Tensor | Int8Tokens", dtype: torch.dtype | None = None) -> torch.Tensor:
        """``xs`` [.., k], values or tokens quantised before; the output is of ``dtype``, by default that of the values."""
        dev = self.device
        t, x, stride, codes, scales, m, out, dtype, _held = _input(xs, self._k, self._n, dev, dtype)
        y = torch.empty(*xs.shape[:-1], self._n, dtype=dtype, device=dev)
        if m:
            _lib.check(_lib.lib().lbq_i8_linear(self._ctx, t, x, stride, codes, scales, m, self._k, self._list, 1, out,
                                                _ADDRESSES[1](y.data_ptr()), _stream(dev)))
        return y

    __call__ = forward

    def __repr__(self) -> str:
        return f"Int8Linear({self.weight!r}, bias={self.bias is not None})"


def _input(xs, k: int, channels: int, device, dtype):
    """(type id, values, stride, codes, scales, rows, out type id, out dtype, what keeps the codes' memory) of a product's
    input."""
    shape, own = xs.shape, xs.dtype
    if not shape or shape[-1] != k:
        raise ValueError(f"input {tuple(shape)} incompatible with k = {k}")
    if xs.device != device:
        raise ValueError(f"input on {xs.device}, weights on {device}")
    if dtype is None:
        dtype = own
    out = _DTYPES.get(dtype)
    if out is None:
        raise ValueError(f"outputs must be f32, f16 or bf16, got {dtype}")
    if isinstance(xs, Int8Tokens):
        return 0, None, 0, xs._rows.data_ptr(), xs.scales.data_ptr(), xs._rows.shape[0], out, dtype, xs
    t, m, stride = _values("the input", xs)
    if m <= _FUSED_ROWS and (m if m < 3 else 4) * _row(k) <= _FUSED_CODES and channels <= _FUSED_CHANNELS:
        return t, xs.data_ptr(), stride, None, None, m, out, dtype, None
    # codes and, behind them, scales
    codes = torch.empty(m * (_row(k) + 4), dtype=torch.int8, device=device)
    at = codes.data_ptr()
    return t, xs.data_ptr(), stride, at, at + m * _row(k), m, out, dtype, codes


def int8_linear_group(linears, xs: "torch.Tensor | Int8Tokens", dtype: torch.dtype | None = None) -> list[torch.Tensor]:
    """``[l.forward(xs, dtype) for l in linears]`` of up to four linears of one k in one call: the input is quantised
    once, and one launch forms the products; the same bits."""
    linears = tuple(linears)
    count = len(linears)
    if not 1 <= count <= GROUP_MAX:
        raise ValueError(f"between 1 and {GROUP_MAX} linears per group, got {count}")
    first = linears[0]
    k, dev = first._k, first.device
    for lin in linears:
        if lin._k != k or lin.device != dev:
            raise ValueError(f"grouped linears must share k and device: {lin._k} on {lin.device}, {k} on {dev}")
    t, x, stride, codes, scales, m, out, dtype, _held = _input(xs, k, sum([lin._n for lin in linears]), dev, dtype)
    lead = xs.shape[:-1]
    ys = [torch.empty(*lead, lin._n, dtype=dtype, device=dev) for lin in linears]
    if m:
        pack = _ADDRESSES[count]
        _lib.check(_lib.lib().lbq_i8_linear(first._ctx, t, x, stride, codes, scales, m, k, pack(*[lin._at for lin in linears]), count, out,
                                            pack(*[y.data_ptr() for y in ys]), _stream(dev)))
    return ys


def int8_gate_up_silu(gate: Int8Linear, up: Int8Linear, xs: "torch.Tensor | Int8Tokens", dtype: torch.dtype | None = None) -> torch.Tensor:
    """``silu(gate(xs)) * up(xs)`` (src/model/mlp_wrapper.rs:190-194) in one call: both products are f32, and neither is
    written."""
    k, dev = gate._k, gate.device
    if up._k != k or up._n != gate._n or up.device != dev:
        raise ValueError(f"gate {gate.weight.shape()} on {dev} and up {up.weight.shape()} on {up.device} must share shape and device")
    t, x, stride, codes, scales, m, out, dtype, _held = _input(xs, k, 2 * gate._n, dev, dtype)
    y = torch.empty(*xs.shape[:-1], gate._n, dtype=dtype, device=dev)
    if m:
        _lib.check(_lib.lib().lbq_i8_gate_up_silu(gate._ctx, t, x, stride, codes, scales, m, k, gate._at, up._at, out, y.data_ptr(), _stream(dev)))
    return y


# ---------------------------------------------------------------------------
# norms
# ---------------------------------------------------------------------------
class Norm(_Fixed):
    """A norm over the last dimension: with u the row (``kind="rms"``), or the row less its mean (``"layer"``),
    ``u / sqrt(mean(u^2) + eps) * (weight + offset) + bias``.  weight and bias are f32 [k]."""

    def __init__(self, weight: torch.Tensor, eps: float, bias: torch.Tensor | None = None, kind: str = "rms", offset: float = 0.0):
        if kind not in _KINDS:
            raise ValueError(f"norm kind {kind!r} is none of {tuple(_KINDS)}")
        k = weight.numel()
        if not 1 <= k <= NORM_MAX_K:
            raise ValueError(f"a norm over {k} values; 1 to {NORM_MAX_K} are served")
        _vector("the norm's weight", weight, k, weight.device)
        if bias is not None:
            _vector("the norm's bias", bias, k, weight.device)
        if not eps >= 0:
            raise ValueError(f"eps = {eps}")
        arg = _lib.NormStruct(_KINDS[kind], eps, offset, weight.data_ptr(), bias.data_ptr() if bias is not None else None)
        vars(self).update(weight=weight, eps=float(eps), bias=bias, kind=kind, offset=float(offset), device=weight.device, _k=k, _arg=arg,
                          _at=ctypes.addressof(arg))


def residual_norm(xs: torch.Tensor, residual: torch.Tensor | None = None, *, post: Norm | None = None, gate: torch.Tensor | None = None,
                  scale: float = 1.0, norm: Norm | None = None, quantize: bool = False) -> "tuple[torch.Tensor, torch.Tensor | Int8Tokens | None]":
    """The residual stream's update by a block's output, and the norm in front of the next block:
    ``r = residual + scale * gate * post(xs)`` and ``y = norm(r)``.

    ``residual`` has the shape of ``xs`` [.., k] and any of the types (its own is r's); ``gate`` is [k] or of the shape of
    ``xs``, and of its type.  What is None is left out; r is ``xs`` itself where nothing is done to it.  y is of ``xs``'s type,
    ``Int8Tokens`` with ``quantize``, None without ``norm``.  Sums over a row are in 64 bits, values in 32, or 64 with
    ``quantize``; y is the norm of r before r is rounded to its type."""
    t, m, stride = _values("xs", xs)
    shape, dev, dtype = xs.shape, xs.device, xs.dtype
    k = shape[-1]
    for n in (post, norm):
        if n is not None and (n._k != k or n.device != dev):
            raise ValueError(f"a norm over {n._k} values on {n.device}, input {tuple(shape)} on {dev}")
    if quantize and norm is None:
        raise ValueError("codes are the norm's result: quantize needs a norm")
    r, rt, rp, rs, gp, gs = xs, t, None, 0, None, 0
    changed = True
    if residual is not None:
        if residual.shape != shape or residual.device != dev:
            raise ValueError(f"residual {tuple(residual.shape)} on {residual.device}, input {tuple(shape)} on {dev}")
        rt, _, rs = _values("the residual", residual)
        rp = residual.data_ptr()
    else:
        changed = gate is not None or post is not None or scale != 1.0
    if gate is not None:
        if gate.dtype != dtype or gate.device != dev:
            raise ValueError(f"gate of {gate.dtype} on {gate.device}, input {dtype} on {dev}")
        if gate.shape == shape:
            _, _, gs = _values("the gate", gate)
        elif gate.shape != shape[-1:] or not gate.is_contiguous():
            raise ValueError(f"gate {tuple(gate.shape)} for input {tuple(shape)}: one contiguous row, or the input's shape")
        gp = gate.data_ptr()
    if changed:
        like, apart = (xs, stride) if residual is None else (residual, rs)
        r = torch.empty_like(like) if apart == k else torch.empty(*shape, dtype=like.dtype, device=dev)
    y = yp = cp = sp = None
    if quantize:
        rows, scales = _empty_tokens(shape, m, dev)
        y, cp, sp = Int8Tokens(rows, scales, shape, dtype, dev), rows.data_ptr(), scales.data_ptr()
    elif norm is not None:
        y = torch.empty_like(xs) if stride == k else torch.empty(*shape, dtype=dtype, device=dev)
        yp = y.data_ptr()
    if m and (changed or norm is not None):
        _lib.check(_lib.lib().lbq_residual_norm(
            _context(dev), t, xs.data_ptr(), stride, rt, rp, rs, None if post is None else post._at, gp, gs, scale,
            None if norm is None else norm._at, m, k, r.data_ptr() if changed else None, yp, cp, sp, _stream(dev)))
    return r, y
