"""Microscaled operators over the gfx950 C ABI: rows and weights in 8 or 4 bits for the scaled matrix
cores, beside :mod:`ancha_amd.fused` (no counterpart in the reference).

Values in blocks of 32 along a row share a power of two and are held as e4m3 codes (``"fp8"``, 8.25 bits
a value) or e2m1 codes (``"fp4"``, 4.25 bits). A RoFormer feed-forward on them::

    up, down = mx.weight(w_in), mx.weight(w_out)        # once, [k, m] float weights
    y, stream = mx.add_unit_norm(x, residual, scale)    # the next layer's input, the residual stream
    hidden = mx.linear(y, up, fused.Epilogue(bias=b_in, gelu=True), format="fp8")
    out = mx.linear(hidden, down, fused.Epilogue(bias=b_out, residual=stream), dtype=stream.dtype)

As in :mod:`ancha_amd.fused`, calls run on the current stream, an op returns ``None`` where the shape or
the device is outside what the kernels cover, and a broken contract raises ``ValueError``. Tensors are
float32, float16 or bfloat16 in any row layout; nothing here is differentiable.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence

import torch

from . import _native
from ._tensors import require, require_optional
from .fused import ATTENTION_HEAD_DIM, Epilogue, _ptr, _stream, _usable

BLOCK = 32
_FORMATS = {"fp8": 8, "fp4": 4}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _format(name: str) -> int:
    if name not in _FORMATS:
        raise ValueError(f"format must be one of {tuple(_FORMATS)}, got {name!r}")
    return _FORMATS[name]


def _type(dtype: torch.dtype, what: str) -> int:
    if dtype not in _TYPES:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {dtype}")
    return _TYPES[dtype]


def _on(device: torch.device):
    """The device of a call's tensors as the current one."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _bytes(t: torch.Tensor, name: str, shape: Sequence[int], align: int) -> torch.Tensor:
    require(t, name, t.device, shape, torch.uint8)
    t = t.contiguous()
    return t if t.data_ptr() % align == 0 else t.clone()


class Tensor:
    """Rows of ``shape[-1]`` values in microscaled form. ``codes`` [rows, pitch] and ``scales``
    [rows, blocks] are uint8 tensors whose rows hold whole groups of 128 values: ``pitch`` is 128 bytes
    a group for "fp8", 64 for "fp4" (two values to a byte, the first in the low half), ``blocks`` 4 a
    group; codes behind ``shape[-1]`` are zero. A scale byte s stands for 2**(s - 127), 255 makes its
    block NaN."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, format: str, shape: Sequence[int]):
        bits = _format(format)
        self.shape = torch.Size(shape)
        if not self.shape:
            raise ValueError("a microscaled tensor has at least one axis")
        rows, groups = self.shape[:-1].numel(), -(-self.shape[-1] // 128)
        for t in (codes, scales):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise ValueError("codes and scales must be tensors on a GPU")
        self.codes = _bytes(codes, "codes", (rows, groups * 16 * bits), 16)
        require(scales, "scales", codes.device, (rows, groups * 4), torch.uint8)
        self.scales = _bytes(scales, "scales", (rows, groups * 4), 4)
        self.format = format

    @classmethod
    def _empty(cls, shape: Sequence[int], format: str, device: torch.device) -> "Tensor":
        self = cls.__new__(cls)
        self.shape, self.format = torch.Size(shape), format
        rows, groups = self.rows, -(-self.shape[-1] // 128)
        self.codes = torch.empty((rows, groups * 16 * _FORMATS[format]), dtype=torch.uint8, device=device)
        self.scales = torch.empty((rows, groups * 4), dtype=torch.uint8, device=device)
        return self

    @property
    def rows(self) -> int:
        return self.shape[:-1].numel()

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def values(self, dtype: torch.dtype = torch.float32) -> Optional[torch.Tensor]:
        """The values that the codes stand for, ``shape`` in ``dtype`` (16 bits hold all but those at
        the ends of the type's range)."""
        kind = _type(dtype, "dtype")
        if not _usable():
            return None
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with _on(self.device):
            rc = _native.lib().ancha_hip_mx_values(
                self.codes.data_ptr(), self.scales.data_ptr(), self.rows, self.shape[-1],
                _FORMATS[self.format], kind, out.data_ptr(), _stream())
        return out if _native.check(rc) else None


class Weight:
    """A [k, m] weight in e2m1 along k, laid out for the matrix cores; made by :func:`weight`."""

    def __init__(self, data: torch.Tensor, k: int, m: int):
        self._data, self.shape = data, torch.Size((k, m))

    @property
    def device(self) -> torch.device:
        return self._data.device

    def values(self, dtype: torch.dtype = torch.float32) -> Optional[torch.Tensor]:
        """The values that the codes stand for, [k, m] in ``dtype``."""
        kind = _type(dtype, "dtype")
        if not _usable():
            return None
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with _on(self.device):
            rc = _native.lib().ancha_hip_mx_weight_values(
                self._data.data_ptr(), *self.shape, kind, out.data_ptr(), _stream())
        return out if _native.check(rc) else None


def _flat(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, dim] with neighbouring columns (a view where its layout allows one)."""
    flat = t if t.dim() == 2 else t.reshape(-1, t.shape[-1]) if t.numel() else \
        t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if flat.shape[0] > 1 and flat.stride(0) < flat.shape[1] or flat.shape[1] > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    return flat


def _stride(flat: torch.Tensor) -> int:
    return max(flat.stride(0), flat.shape[1]) if flat.shape[0] > 1 else flat.shape[1]


def _rows_op(x: torch.Tensor, name: str) -> Optional[int]:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a tensor on a GPU")
    if x.dim() == 0:
        raise ValueError(f"{name} must have at least one axis")
    return _type(x.dtype, name) if _usable() else None


def quantize(x: torch.Tensor, format: str = "fp4") -> Optional[Tensor]:
    """``x`` [..., dim] in blocks of 32 along its last axis."""
    bits, kind = _format(format), _rows_op(x, "x")
    if kind is None:
        return None
    flat = _flat(x)
    out = Tensor._empty(x.shape, format, x.device)
    with _on(x.device):
        rc = _native.lib().ancha_hip_mx_quantize(
            flat.data_ptr(), kind, flat.shape[0], flat.shape[1], _stride(flat), bits,
            out.codes.data_ptr(), out.scales.data_ptr(), _stream())
    return out if _native.check(rc) else None


def _norm(x, residual, scale, eps, format):
    bits, kind = _format(format), _rows_op(x, "x")
    if kind is None:
        return None, None
    dim = x.shape[-1]
    require_optional(scale, "scale", x.device, (dim,))
    flat, total, other = _flat(x), None, None
    if residual is not None:
        require(residual, "residual", x.device, x.shape, x.dtype)
        other = _flat(residual)
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out = Tensor._empty(x.shape, format, x.device)
    s = None if scale is None else scale.contiguous()
    with _on(x.device):
        rc = _native.lib().ancha_hip_mx_norm(
            flat.data_ptr(), kind, flat.shape[0], dim, _stride(flat), _ptr(other),
            0 if other is None else _stride(other), _ptr(s), float(eps), bits, _ptr(total),
            out.codes.data_ptr(), out.scales.data_ptr(), _stream())
    return (out, total) if _native.check(rc) else (None, None)


def unit_norm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, eps: float = 0.0,
              format: str = "fp8") -> Optional[Tensor]:
    """``x * scale / max(sqrt(sum x^2 + dim * eps), 1e-12)`` over the last axis of ``x`` [..., dim], in
    blocks of 32: :func:`ancha_amd.fused.unit_norm` with codes for its output, and with
    ``scale = sqrt(dim) * gamma`` and ``eps`` > 0 the root-mean-square norm. Evaluated in 64 bits, so
    the only rounding is the one to the codes."""
    return _norm(x, None, scale, eps, format)[0]


def add_unit_norm(x: torch.Tensor, residual: torch.Tensor, scale: Optional[torch.Tensor] = None,
                  eps: float = 0.0, format: str = "fp8") -> Optional[tuple[Tensor, torch.Tensor]]:
    """:func:`unit_norm` of ``x + residual`` (same shape and type; the sum is rounded to that type)
    and the sum itself, the residual stream that goes on."""
    if residual is None:
        raise ValueError("residual must be a torch tensor")
    out, total = _norm(x, residual, scale, eps, format)
    return None if out is None else (out, total)


def weight(w: torch.Tensor) -> Optional[Weight]:
    """The [k, m] weight ``w`` (Burn Linear layout as in :func:`ancha_amd.fused.linear`; the transposed
    view of a PyTorch [out, in] weight is as good) in e2m1 with blocks of 32 along k. Made once, when a
    model is loaded."""
    kind = _rows_op(w, "w")
    if w.dim() != 2:
        raise ValueError(f"w must be [k, m], got {tuple(w.shape)}")
    if kind is None:
        return None
    k, m = w.shape
    size = int(_native.lib().ancha_hip_mx_weight_bytes(k, m))
    if size == 0:
        return None
    if min(w.stride()) < 0 or (0 in w.stride()):
        w = w.contiguous()
    data = torch.empty(size, dtype=torch.uint8, device=w.device)
    with _on(w.device):
        rc = _native.lib().ancha_hip_mx_weight(w.data_ptr(), kind, k, m, *w.stride(), data.data_ptr(),
                                               _stream())
    return Weight(data, k, m) if _native.check(rc) else None


def linear(x: Tensor, w: Weight, epilogue: Optional[Epilogue] = None,
           dtype: torch.dtype = torch.float32, format: Optional[str] = None):
    """``x`` [..., k] . ``w`` [k, m] through the epilogue of :func:`ancha_amd.fused.linear` (bias ->
    erf-GELU -> rotary -> residual; bias and rotary table float32, the residual [..., m] in ``dtype``):
    [..., m] in ``dtype``, or with ``format`` the :class:`Tensor` of the float32 result, the next
    product's operand. Any k, m > 0; ``None`` for an empty axis or a rotary shape that does not fit.

    Products of codes are exact and sums are held in 32 bits; "fp8" rows with a 16-bit ``dtype`` take
    the matrix cores' shorter sums (4e-6 of the result on normal data, far below the type's step)."""
    if not isinstance(x, Tensor) or not isinstance(w, Weight):
        raise ValueError("linear takes a microscaled Tensor and a Weight")
    e = epilogue or Epilogue()
    kind = _type(dtype, "dtype")
    bits = 0 if format is None else _format(format)
    if bits and dtype != torch.float32:
        raise ValueError("an output in codes is taken from the float32 result: leave dtype alone")
    n, (k, m) = x.rows, w.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has rows of {x.shape[-1]}, the weight takes {k}")
    if w.device != x.device:
        raise ValueError(f"the weight must be on {x.device}, got {w.device}")
    shape = x.shape[:-1] + (m,)
    tokens = width = 0
    table = None
    if e.rotary is not None:
        table, width = e.rotary
        require(table, "rotary table", x.device)
        if table.dim() != 3 or table.shape[0] != 4 or table.shape[2] != ATTENTION_HEAD_DIM:
            return None
        tokens = table.shape[1]
        if tokens == 0 or n % tokens or width < 0 or width % 64 or 2 * width > m:
            return None
        table = table.contiguous()
    require_optional(e.bias, "bias", x.device, (m,))
    require_optional(e.residual, "residual", x.device, shape, dtype)
    bias = None if e.bias is None else e.bias.contiguous()
    residual = None if e.residual is None else e.residual.contiguous()
    if not _usable():
        return None
    if bits:
        out = Tensor._empty(shape, format, x.device)
        to, scales = out.codes.data_ptr(), out.scales.data_ptr()
    else:
        out = torch.empty(shape, dtype=dtype, device=x.device)
        to, scales = out.data_ptr(), None
    with _on(x.device):
        rc = _native.lib().ancha_hip_mx_linear(
            x.codes.data_ptr(), x.scales.data_ptr(), n, k, _FORMATS[x.format], w._data.data_ptr(), m,
            _ptr(bias), int(e.gelu), _ptr(table), tokens, width, _ptr(residual), kind, bits, to, scales,
            _stream())
    return out if _native.check(rc) else None
