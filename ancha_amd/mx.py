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

from typing import Optional, Sequence

import torch

from . import _native
from ._tensors import require
from .fused import ATTENTION_HEAD_DIM, Epilogue, _ptr

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


def _launch(index: int, name: str, *args) -> bool:
    """Entry point ``name`` on the current stream of GPU ``index``, the one its tensors are on."""
    fn = getattr(_native.lib(), name)
    if index == torch._C._cuda_getDevice():
        return _native.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))
    with torch.cuda.device(index):
        return _native.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))


def _bytes(t: torch.Tensor, name: str, device: torch.device, shape: Sequence[int],
           align: int) -> torch.Tensor:
    require(t, name, device, shape, torch.uint8)
    t = t.contiguous()
    return t if t.data_ptr() % align == 0 else t.clone()


class Tensor:
    """Rows of ``shape[-1]`` values in microscaled form. ``codes`` [rows, pitch] and ``scales``
    [rows, blocks] are uint8 tensors whose rows hold whole groups of 128 values: ``pitch`` is 128 bytes
    a group for "fp8", 64 for "fp4" (two values to a byte, the first in the low half), ``blocks`` 4 a
    group; behind ``shape[-1]`` codes are zero and scales not 255. A scale byte s stands for
    2**(s - 127), 255 makes its block NaN."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, format: str, shape: Sequence[int]):
        bits = _format(format)
        self.shape, self.format = torch.Size(shape), format
        if not self.shape:
            raise ValueError("a microscaled tensor has at least one axis")
        for t in (codes, scales):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise ValueError("codes and scales must be tensors on a GPU")
        self.rows, groups = self.shape[:-1].numel(), -(-self.shape[-1] // 128)
        self._codes = _bytes(codes, "codes", codes.device, (self.rows, groups * 16 * bits), 16)
        self._scales = _bytes(scales, "scales", codes.device, (self.rows, groups * 4), 4)
        self._whole = None

    @classmethod
    def _empty(cls, shape: torch.Size, rows: int, format: str, device: torch.device) -> "Tensor":
        """Room for ``rows`` rows, codes and scales in one allocation."""
        self = cls.__new__(cls)
        self.shape, self.rows, self.format = shape, rows, format
        self._codes = self._scales = None
        self._whole = torch.empty(rows * -(-shape[-1] // 128) * (16 * _FORMATS[format] + 4),
                                  dtype=torch.uint8, device=device)
        return self

    def _split(self) -> int:
        return self.rows * -(-self.shape[-1] // 128) * 16 * _FORMATS[self.format]

    def _pointers(self) -> tuple[int, int]:
        if self._whole is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        at = self._whole.data_ptr()
        return at, at + self._split()

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._whole[:self._split()].view(
                self.rows, -(-self.shape[-1] // 128) * 16 * _FORMATS[self.format])
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._whole[self._split():].view(self.rows, -(-self.shape[-1] // 128) * 4)
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._codes if self._whole is None else self._whole).device

    def values(self, dtype: torch.dtype = torch.float32) -> Optional[torch.Tensor]:
        """The values that the codes stand for, ``shape`` in ``dtype`` (16 bits hold all but those at
        the ends of the type's range)."""
        kind = _type(dtype, "dtype")
        device = self.device
        out = torch.empty(tuple(self.shape), dtype=dtype, device=device)
        codes, scales = self._pointers()
        return out if _launch(device.index, "ancha_mx_values", codes, scales, self.rows,
                              self.shape[-1], _FORMATS[self.format], kind, out.data_ptr()) else None


class Weight:
    """A [k, m] weight in e2m1 along k, laid out for the matrix cores; made by :func:`weight`. ``data`` is the
    uint8 tensor that such a weight of the same shape holds."""

    def __init__(self, data: torch.Tensor, k: int, m: int):
        size = int(_native.lib().ancha_mx_weight_bytes(k, m)) if k > 0 and m > 0 else 0
        if size == 0:
            raise ValueError(f"no weight has the shape [{k}, {m}]")
        if not isinstance(data, torch.Tensor) or not data.is_cuda:
            raise ValueError("data must be a tensor on a GPU")
        self._data, self.shape = _bytes(data, "data", data.device, (size,), 16), torch.Size((k, m))

    @property
    def device(self) -> torch.device:
        return self._data.device

    def values(self, dtype: torch.dtype = torch.float32) -> Optional[torch.Tensor]:
        """The values that the codes stand for, [k, m] in ``dtype``."""
        kind = _type(dtype, "dtype")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        return out if _launch(self.device.index, "ancha_mx_weight_values", self._data.data_ptr(),
                              *self.shape, kind, out.data_ptr()) else None


def _rows(t: torch.Tensor, dim: int, rows: int) -> tuple[torch.Tensor, int]:
    """t [..., dim] as ``rows`` rows of neighbouring columns (a view where its layout allows one) and
    their stride."""
    if t.is_contiguous():
        return t, dim
    flat = t if t.dim() == 2 else t.reshape(rows, dim)
    stride = flat.stride()
    if (rows > 1 and stride[0] < dim) or (dim > 1 and stride[1] != 1):
        return flat.contiguous(), dim
    return flat, stride[0] if rows > 1 else dim


def _input(x: torch.Tensor, name: str) -> int:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a tensor on a GPU")
    if x.dim() == 0:
        raise ValueError(f"{name} must have at least one axis")
    return _type(x.dtype, name)


def quantize(x: torch.Tensor, format: str = "fp4") -> Optional[Tensor]:
    """``x`` [..., dim] in blocks of 32 along its last axis."""
    bits, kind = _format(format), _input(x, "x")
    shape = x.shape
    dim = shape[-1]
    rows = shape[:-1].numel()
    flat, ld = _rows(x, dim, rows)
    out = Tensor._empty(shape, rows, format, x.device)
    codes, scales = out._pointers()
    return out if _launch(x.get_device(), "ancha_mx_quantize", flat.data_ptr(), kind, rows, dim, ld,
                          bits, codes, scales) else None


def _norm(x, residual, scale, eps, format):
    bits, kind = _format(format), _input(x, "x")
    shape, device = x.shape, x.device
    dim = shape[-1]
    rows = shape[:-1].numel()
    if scale is not None:
        require(scale, "scale", device, (dim,))
        scale = scale.contiguous()
    flat, ld = _rows(x, dim, rows)
    total, ldr = None, 0
    if residual is not None:
        require(residual, "residual", device, shape, x.dtype)
        residual, ldr = _rows(residual, dim, rows)
        total = torch.empty_like(x, memory_format=torch.contiguous_format)
    out = Tensor._empty(shape, rows, format, device)
    codes, scales = out._pointers()
    done = _launch(device.index, "ancha_mx_norm", flat.data_ptr(), kind, rows, dim, ld, _ptr(residual),
                   ldr, _ptr(scale), float(eps), bits, _ptr(total), codes, scales)
    return (out, total) if done else (None, None)


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
    kind = _input(w, "w")
    if w.dim() != 2:
        raise ValueError(f"w must be [k, m], got {tuple(w.shape)}")
    k, m = w.shape
    size = int(_native.lib().ancha_mx_weight_bytes(k, m))
    if size == 0:
        return None
    if min(w.stride()) < 0 or (0 in w.stride()):
        w = w.contiguous()
    data = torch.empty(size, dtype=torch.uint8, device=w.device)
    return Weight(data, k, m) if _launch(w.get_device(), "ancha_mx_weight", w.data_ptr(), kind, k, m,
                                         *w.stride(), data.data_ptr()) else None


def linear(x: Tensor, w: Weight, epilogue: Optional[Epilogue] = None,
           dtype: torch.dtype = torch.float32, format: Optional[str] = None):
    """``x`` [..., k] . ``w`` [k, m] through the epilogue of :func:`ancha_amd.fused.linear` (bias ->
    erf-GELU -> rotary -> residual; bias and rotary table float32, the residual [..., m] in ``dtype``):
    [..., m] in ``dtype``, or with ``format`` the :class:`Tensor` of the float32 result, the next
    product's operand. Any k, m > 0; ``None`` for an empty axis or a rotary shape that does not fit.

    Products of codes are exact and sums are held in 32 bits, whatever ``dtype`` ("fp8" rows take the
    matrix cores two passes for that, so twice the time of "fp4" rows where these are what bounds). GELU is
    off by at most 4e-6 of its value for arguments above -4 and 2e-3 below (16-bit results and codes: 3e-5,
    3e-3). The order of a row's sums depends on n, k and m, so its last bits may differ from one n to another."""
    if not isinstance(x, Tensor) or not isinstance(w, Weight):
        raise ValueError("linear takes a microscaled Tensor and a Weight")
    kind = _type(dtype, "dtype")
    bits = 0 if format is None else _format(format)
    if bits and dtype != torch.float32:
        raise ValueError("an output in codes is taken from the float32 result: leave dtype alone")
    n, device, (k, m) = x.rows, x.device, w.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has rows of {x.shape[-1]}, the weight takes {k}")
    if w.device != device:
        raise ValueError(f"the weight must be on {device}, got {w.device}")
    shape = x.shape[:-1] + (m,)
    bias = residual = table = None
    gelu = tokens = width = 0
    if epilogue is not None:
        bias, residual, gelu = epilogue.bias, epilogue.residual, int(epilogue.gelu)
        if epilogue.rotary is not None:
            table, width = epilogue.rotary
            require(table, "rotary table", device)
            if table.dim() != 3 or table.shape[0] != 4 or table.shape[2] != ATTENTION_HEAD_DIM:
                return None
            tokens = table.shape[1]
            if tokens == 0 or n % tokens or width < 0 or width % 64 or 2 * width > m:
                return None
            table = table.contiguous()
        if bias is not None:
            require(bias, "bias", device, (m,))
            bias = bias.contiguous()
        if residual is not None:
            require(residual, "residual", device, shape, dtype)
            residual = residual.contiguous()
    if bits:
        out = Tensor._empty(shape, n, format, device)
        to, to_scales = out._pointers()
    else:
        out = torch.empty(tuple(shape), dtype=dtype, device=device)
        to, to_scales = out.data_ptr(), None
    codes, scales = x._pointers()
    return out if _launch(device.index, "ancha_mx_linear", codes, scales, n, k, _FORMATS[x.format],
                          w._data.data_ptr(), m, _ptr(bias), gelu, _ptr(table), tokens, width,
                          _ptr(residual), kind, bits, to, to_scales) else None
