"""ancha_amd: the MI355X-native (gfx950) fused RoFormer attention path of Ancha.

The compute lives in hand-written HIP kernels behind the C ABI of ``include/ancha_hip.h``
(``ancha_amd/_lib/libancha_hip.so``); :mod:`ancha_amd.fused` mirrors the reference's
``ancha_models::fused`` op boundary on top of it, and :mod:`ancha_amd.mx` has the same kind of ops on
8- and 4-bit microscaled operands. :mod:`ancha_amd.paged` adds what serving token by token needs between them:
rotary positions, a paged cache in those codes and attention over it.
"""
from . import fused, mx, paged  # noqa: F401
from ._native import HipError, LIB_PATH, build  # noqa: F401

__all__ = ["fused", "mx", "paged", "HipError", "LIB_PATH", "build"]
