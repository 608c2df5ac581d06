"""Attention over a paged cache where its numbers are at their limits, against the 64-bit oracle: values and NaN in the
cache of any size. Both kernels, tiles and chunks.
"""
import numpy as np
import pytest
import torch

from ancha_amd import paged
from ancha_amd import workload as W
from oracle import paged as O
from tests.test_paged_gpu import CHUNK, TYPES, dev, form, host, some_batch, some_cache

pytestmark = pytest.mark.gpu

FORMS = [(4, None), (20, 9000)]  # heads over 2 of the cache, columns of the table: tiles and chunks


def on(gpu, codes, scales, fmt):
    return paged.Cache(torch.from_numpy(codes.copy()).to(gpu), torch.from_numpy(scales.copy()).to(gpu), fmt)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,columns", FORMS)
def test_a_nan_is_seen_behind_the_largest_values(gpu, heads, columns, kind):
    """Finite values of 2^126 and more in 4 bits (scale byte 252), and a NaN in a later step that has nothing else."""
    cache, codes, scales = some_cache(gpu, 8, 64, 2, 64, "fp4", 201)
    batch, plain, rows = some_batch(gpu, [230], [230], 64, 8, 202, columns=columns)
    assert (form(kind, rows, heads, cache, batch)[0] == CHUNK) == bool(columns)
    k, v = (dev(W.normal((rows, 2, 64), s, 1.0), gpu) for s in (203, 204))
    v[3, :, 32:], v[150, 1, 40] = 2.4e38, float("nan")
    assert cache.write(k, v, batch) is cache
    O.write(codes, scales, "fp4", host(k), host(v), plain)
    assert np.array_equal(cache.scales.cpu().numpy(), scales) and scales.max() == 255 and (scales == 252).any()
    q = dev(W.normal((rows, heads, 64), 205, 1.0), gpu, TYPES[kind])
    got = torch.isnan(paged.attention(q, cache, batch)).cpu().numpy()
    want = np.zeros(got.shape, bool)
    want[150:, heads // 2:, 32:] = True
    assert np.array_equal(got, want), f"NaN in {got.sum()} places, not {want.sum()}"


@pytest.mark.parametrize("heads,columns", FORMS)
@pytest.mark.parametrize("byte", [248, 252, 254])
def test_a_nan_is_seen_behind_any_scale(gpu, byte, heads, columns):
    """A caller's own e4m3 codes: ones under the largest scales, then a NaN block alone in its step."""
    cache, codes, scales = some_cache(gpu, 8, 64, 2, 64, "fp8", 211)
    batch, plain, rows = some_batch(gpu, [230], [230], 64, 8, 212, columns=columns)
    for t, s, code in ((3, byte, 0x38), (150, 255, 0)):
        page, slot = O.place(plain, 0, t, 8, 64)
        scales[1, page, 1, slot, 0], codes[1, page, 1, slot, :32] = s, code
    cache = on(gpu, codes, scales, "fp8")
    q = dev(W.normal((rows, heads, 64), 213, 1.0), gpu, torch.bfloat16)
    got = torch.isnan(paged.attention(q, cache, batch)).cpu().numpy()
    want = np.zeros(got.shape, bool)
    want[150:, heads // 2:, :32] = True
    assert np.array_equal(got, want), f"NaN in {got.sum()} places, not {want.sum()}"
