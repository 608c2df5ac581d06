"""Serving token by token over the gfx950 C ABI, beside :mod:`ancha_amd.mx` (no counterpart in the reference): rotary
positions, a cache of keys and values in pages of microscaled codes, and attention of new tokens over it.

One layer's attention for the new tokens of some sequences, one each or whole prompts, rows beside each other::

    plan = paged.rotary_plan(128, base=500000.0, scaling="yarn", factor=16.0, original=8192)   # once
    cache = paged.Cache.empty(pages, 64, kv_heads, 128, "fp8")                                 # once a layer
    batch = paged.Batch(starts, lengths, table)                                               # once a step
    qkv = mx.linear(x, w_qkv, dtype=torch.bfloat16).view(-1, heads + 2 * kv_heads, 128)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    cache.write(k, v, batch, plan)                          # keys are rotated as they are written
    out = paged.attention(paged.rotary(q, batch, plan), cache, batch)

As in :mod:`ancha_amd.mx`, calls run on the current stream, an op returns ``None`` where the shape or the device is
outside what the kernels cover, and a broken contract raises ``ValueError``. Tensors are float32, float16 or bfloat16
in any row layout; nothing here is differentiable. What a batch holds is read on the GPU, when the kernels run, so a
captured step is replayed on new lengths and pages by writing them into the same tensors; the kernels check every row
and page number that they find there.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Union

import torch

from . import _native
from ._tensors import require
from .mx import BLOCK, _format, _input, _launch, _type

DIMS = (64, 128, 256)
_LAYOUTS = ("half", "interleaved")


def _whole(t: torch.Tensor, name: str, dtype: torch.dtype, dims: int) -> torch.Tensor:
    """A contiguous GPU tensor, kept as it is: it is read, or written, in place later."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on a GPU")
    if t.dtype != dtype or t.dim() != dims:
        raise ValueError(f"{name} must be {dtype} with {dims} axes, got {t.dtype} {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


class Batch:
    """Sequences of a call, int32 tensors on the GPU. The rows ``starts[i]`` to ``starts[i + 1]`` (ascending,
    [sequences + 1]) are new tokens of sequence i, which has ``lengths[i]`` tokens with them, so the last row is at
    position ``lengths[i] - 1``; token t lies in page ``table[i, t // page]`` ([sequences, columns]). A number outside
    the cache's pages is a page that is not there: its tokens are not seen, not written and read as zeros. Rows behind
    the last sequence (or before the first) are of none."""

    def __init__(self, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor):
        self.starts = _whole(starts, "starts", torch.int32, 1)
        self.lengths = _whole(lengths, "lengths", torch.int32, 1)
        self.table = _whole(table, "table", torch.int32, 2)
        self.device = lengths.device
        count = lengths.shape[0]
        require(starts, "starts", self.device, (count + 1,), torch.int32)
        require(table, "table", self.device, (count, table.shape[1]), torch.int32)
        self._c = _native.PagedBatch(starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), count, table.shape[1])
        self._at = ctypes.addressof(self._c)

    def __len__(self) -> int:
        return self.lengths.shape[0]


class Rotary:
    """Rotary positions, made by :func:`rotary_plan` or of frequencies of one's own: ``freqs`` [width / 2] float64 on
    the GPU, radians a position of each pair, at most 2**20 in magnitude. The first ``width`` columns of a head are
    turned, in pairs (i, i + width / 2) for the layout "half" and (2 i, 2 i + 1) for "interleaved", and multiplied by
    ``magnitude``."""

    def __init__(self, freqs: torch.Tensor, layout: str = "half", magnitude: float = 1.0):
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {_LAYOUTS}, got {layout!r}")
        self.freqs, self.layout, self.magnitude = _whole(freqs, "freqs", torch.float64, 1), layout, float(magnitude)
        if not freqs.shape[0]:
            raise ValueError("freqs must not be empty")
        if not (math.isfinite(self.magnitude) and self.magnitude > 0):
            raise ValueError(f"magnitude must be a number > 0, got {magnitude}")
        self.width, self.device = 2 * freqs.shape[0], freqs.device
        self._c = _native.PagedPlan(freqs.data_ptr(), self.width, int(layout == "interleaved"), self.magnitude)
        self._at = ctypes.addressof(self._c)


def frequencies(width: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                original: int = 0) -> tuple[list[float], float]:
    """(radians a position of each of ``width / 2`` pairs, magnitude): ``base ** (-2 i / width)``, for contexts
    ``factor`` times as long as the model was trained on with ``scaling``

    "linear"  positions divided by ``factor``;
    "ntk"     the base times ``factor ** (width / (width - 2))``: the last pair is slowed down by ``factor``, the
              first not;
    "yarn"    pairs that turn less than once over the ``original`` tokens are slowed down by ``factor``, those that
              turn over 32 times not, those between in proportion to their turns; magnitude ``0.1 ln(factor) + 1``.
              Checkpoints whose ramp goes by the pair's index between two rounded borders instead, as widely used
              loaders have it, need those frequencies: :class:`Rotary` takes any."""
    if width < 2 or width % 2 or not (math.isfinite(base) and base > 0):
        raise ValueError(f"width must be even and > 0 and base a number > 0, got {width} and {base}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if not (math.isfinite(factor) and factor >= 1) or (scaling is None and factor != 1):
        raise ValueError("factor must be a number >= 1, and 1 without scaling")
    if scaling == "ntk":
        if width == 2:
            raise ValueError("'ntk' takes a width above 2")
        # By logarithms, as the power may pass the range of a float.
        if math.log(base) + width / (width - 2) * math.log(factor) >= 709:
            raise ValueError(f"factor {factor} makes a base beyond 64-bit numbers")
        base = base * factor ** (width / (width - 2))
    if math.log2(base) * (2 - width) / width > 20:
        raise ValueError(f"base {base} makes frequencies above 2**20")
    freqs = [base ** (-2 * i / width) for i in range(width // 2)]
    if scaling == "linear":
        return [f / factor for f in freqs], 1.0
    if scaling != "yarn":
        return freqs, 1.0
    if not 1 <= original <= 2 ** 53:
        raise ValueError("'yarn' takes the original length in tokens")
    keep = [min(1.0, max(0.0, (original * f / (2 * math.pi) - 1) / 31)) for f in freqs]
    return [f * (g + (1 - g) / factor) for f, g in zip(freqs, keep)], 0.1 * math.log(factor) + 1


def rotary_plan(width: int, base: float = 10000.0, layout: str = "half", scaling: Optional[str] = None,
                factor: float = 1.0, original: int = 0, device: Union[str, torch.device] = "cuda") -> Rotary:
    """The :class:`Rotary` of :func:`frequencies`, made once, when a model is loaded."""
    freqs, magnitude = frequencies(width, base, scaling, factor, original)
    return Rotary(torch.tensor(freqs, dtype=torch.float64, device=device), layout, magnitude)


_POSITIONS = {torch.int32: 4, torch.int64: 8}


def _take(x: torch.Tensor, name: str) -> int:
    kind = _input(x, name)
    if x.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, dim], got {tuple(x.shape)}")
    return kind


def _strides(x: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """x [rows, heads, dim] with neighbouring columns (a copy where they are not), its strides of rows and heads."""
    row, head, column = x.stride()
    if column == 1 or x.shape[2] == 1:
        return x, row, head
    x = x.contiguous()
    return x, x.stride(0), x.stride(1)


def _on(owner, name: str, kind: type, device: torch.device) -> None:
    if isinstance(owner, kind) and owner.device == device:
        return
    if not isinstance(owner, kind):
        raise ValueError(f"{name} must be a paged.{kind.__name__}")
    raise ValueError(f"{name} must be on {device}, got {owner.device}")


def rotary(x: torch.Tensor, positions: Union[torch.Tensor, Batch], plan: Rotary) -> Optional[torch.Tensor]:
    """``x`` [rows, heads, dim] with each row's heads turned by its position: (x, y) of a pair becomes
    ``magnitude * (x cos a - y sin a, y cos a + x sin a)``, ``a = position * freqs[i]`` in 64 bits, the rest in 32.
    ``positions``: [rows], int32 or int64 (negative ones turn back), or the :class:`Batch` that the rows are of (rows of
    no sequence give zeros)."""
    kind = _take(x, "x")
    device = x.device
    _on(plan, "plan", Rotary, device)
    rows, heads, dim = x.shape
    if plan.width > dim:
        raise ValueError(f"the plan turns {plan.width} columns, x has {dim}")
    at = batch = None
    wide = 0
    if isinstance(positions, Batch):
        _on(positions, "positions", Batch, device)
        batch = positions._at
    else:
        wide = _POSITIONS.get(getattr(positions, "dtype", None), 0)
        if not wide:
            raise ValueError("positions must be an int32 or int64 tensor or a paged.Batch")
        if positions.shape != (rows,) or positions.device != device:
            require(positions, "positions", device, (rows,), positions.dtype)
        positions = positions.contiguous()
        at = positions.data_ptr()
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if not out.numel():
        return out
    x, row, head = _strides(x)
    return out if _launch(device.index, "ancha_paged_rotary", x.data_ptr(), kind, rows, heads, dim, row, head, at, wide,
                          batch, plan._at, out.data_ptr()) else None


class Cache:
    """Keys and values of one layer in pages: uint8 ``codes`` [2, pages, heads, page, dim] (for "fp4" dim / 2, the
    first value in the low half) and ``scales`` [2, pages, heads, page, dim / 32], keys first, by the formats of
    :mod:`ancha_amd.mx` with blocks of 32 along the head. ``page`` tokens a page, a power of two from 16 to 65536;
    ``dim`` 64, 128 or 256. Pages are the caller's: any page may be given to any sequence, be shared by several that
    only read it, or be copied (``cache.codes[:, to] = cache.codes[:, at]``, and the scales). Codes of one's own have to
    be numbers, as :meth:`write` makes them: a NaN is told by its block's scale byte, 255, and e4m3's own NaN codes
    (0x7f and 0xff) among a token's values would reach rows that do not see it."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, format: str):
        bits = _format(format)
        self.codes, self.scales = _whole(codes, "codes", torch.uint8, 5), _whole(scales, "scales", torch.uint8, 5)
        self.format, self.device = format, codes.device
        self.pages, self.heads, self.page = codes.shape[1:4]
        self.dim = codes.shape[4] * 8 // bits
        if codes.shape[0] != 2 or self.dim not in DIMS:
            raise ValueError(f"codes must be [2, pages, heads, page, bytes of {DIMS} values], got {tuple(codes.shape)}")
        if self.page & (self.page - 1) or not 16 <= self.page <= 65536:
            raise ValueError(f"a page holds a power of two of tokens from 16 to 65536, got {self.page}")
        if not self.pages or not self.heads:
            raise ValueError("a cache has at least one page and one head")
        require(scales, "scales", self.device, codes.shape[:4] + (self.dim // BLOCK,), torch.uint8)
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("codes and scales must be 16-byte aligned")
        self._c = _native.PagedCache(codes.data_ptr(), scales.data_ptr(), self.pages, self.heads, self.page, self.dim,
                                     bits)
        self._at = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, pages: int, page: int, heads: int, dim: int, format: str = "fp8",
              device: Union[str, torch.device] = "cuda") -> "Cache":
        """A cache without tokens (all zeros)."""
        bits = _format(format)
        if dim not in DIMS:
            raise ValueError(f"dim must be one of {DIMS}, got {dim}")
        shape = (2, pages, heads, page)
        return cls(torch.zeros(shape + (dim * bits // 8,), dtype=torch.uint8, device=device),
                   torch.zeros(shape + (dim // BLOCK,), dtype=torch.uint8, device=device), format)

    def write(self, k: torch.Tensor, v: torch.Tensor, batch: Batch,
              plan: Optional[Rotary] = None) -> Optional["Cache"]:
        """The rows' keys and values [rows, heads, dim] into the places that ``batch`` gives them, keys first turned by
        ``plan`` where there is one. Rotated in 64 bits, so the rounding to the codes is the only one; a NaN or an
        infinity (2**128 or more) makes its block of 32 NaN. Rows of no sequence, in a page that is not there or at a
        position below 0 are left out. No two rows may have the same place."""
        kind = _take(k, "k")
        require(v, "v", self.device, k.shape, k.dtype)
        if k.device != self.device or k.shape[1:] != (self.heads, self.dim):
            raise ValueError(f"k must be [rows, {self.heads}, {self.dim}] on {self.device}, got {tuple(k.shape)} on "
                             f"{k.device}")
        _on(batch, "batch", Batch, self.device)
        if plan is not None:
            _on(plan, "plan", Rotary, self.device)
            if plan.width > self.dim:
                raise ValueError(f"the plan turns {plan.width} columns, the heads have {self.dim}")
        if not k.numel():
            return self
        k, ldk, ldkh = _strides(k)
        v, ldv, ldvh = _strides(v)
        done = _launch(self.device.index, "ancha_paged_write", k.data_ptr(), v.data_ptr(), kind, k.shape[0], ldk, ldkh,
                       ldv, ldvh, batch._at, None if plan is None else plan._at, self._at)
        return self if done else None

    def read(self, batch: Batch, size: int,
             dtype: torch.dtype = torch.bfloat16) -> Optional[tuple[torch.Tensor, torch.Tensor]]:
        """(keys, values) [sequences, size, heads, dim]: what is held for the tokens 0 to ``size`` of each sequence
        (keys as they were written, rotated), zeros behind its length."""
        kind = _type(dtype, "dtype")
        _on(batch, "batch", Batch, self.device)
        if size < 0:
            raise ValueError(f"size must be >= 0, got {size}")
        k = torch.empty((len(batch), size, self.heads, self.dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if not k.numel():
            return k, v
        return (k, v) if _launch(self.device.index, "ancha_paged_read", self._at, batch._at, size, kind, k.data_ptr(),
                                 v.data_ptr()) else None


def attention(q: torch.Tensor, cache: Cache, batch: Batch, scale: Optional[float] = None, causal: bool = True,
              window: Optional[int] = None) -> Optional[torch.Tensor]:
    """``softmax(scale q.k) v`` of each row of ``q`` [rows, heads, dim] over the cached tokens of its sequence (those of
    this call too, written before it); [rows, heads, dim] in q's type. ``heads`` is a multiple of the cache's: head h
    reads head ``h // (heads // cache.heads)`` of it. A row at position t sees the tokens up to t, or without ``causal``
    all of its sequence (an encoder's states), and with ``window`` none before ``t - window + 1``. Rows that see no
    token and rows of no sequence are 0. ``scale`` > 0 is 1 / sqrt(dim) if not given.

    Scores are exact to 32 bits for every type of q; weights are off by 2**-21 of themselves at most or by 2**-37 of
    their row's largest, and sums are held in 32, so a result is rounded to its type once. Values more than 2**30 below
    the largest of their head's block of 32 columns, of any token that this row or those beside it see, may be rounded.
    A score beyond float32 is infinite: minus infinity weighs nothing, plus infinity makes its row NaN, as does a row of
    nothing but minus infinity. A NaN in the cache (scale byte 255) reaches the rows that see its token, no others. How
    the keys are shared out depends on shapes and lengths alone, so a call gives the same bits
    every time."""
    kind = _take(q, "q")
    device = q.device
    _on(cache, "cache", Cache, device)
    _on(batch, "batch", Batch, device)
    rows, heads, dim = q.shape
    if dim != cache.dim or heads % cache.heads or not heads:
        raise ValueError(f"q must have a multiple of {cache.heads} heads of {cache.dim} columns, got {tuple(q.shape)}")
    if window is not None and window < 1:
        raise ValueError(f"window must be >= 1, got {window}")
    scale = dim ** -0.5 if scale is None else float(scale)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if not rows:
        return out
    q, row, head = _strides(q)
    need = _native.lib().ancha_paged_attention_workspace(kind, rows, heads, cache._at, batch._at)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    return out if _launch(device.index, "ancha_paged_attention", q.data_ptr(), kind, rows, heads, row, head,
                          cache._at, batch._at, scale, int(causal), min(window or 0, 2 ** 31),
                          None if workspace is None else workspace.data_ptr(), need, out.data_ptr()) else None
