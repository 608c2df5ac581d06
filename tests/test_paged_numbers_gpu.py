"""Attention over a paged cache where its numbers are at their limits, against the 64-bit oracle: values and NaN in the
cache of any size, weights to 22 bits and small ones, large and infinite scores,
large queries. Both kernels, tiles and chunks.
"""
import numpy as np
import pytest
import torch

from ancha_amd import paged
from ancha_amd import workload as W
from oracle import mx as OM
from oracle import paged as O
from tests.test_paged_gpu import CHUNK, PARTS, TYPES, close, dev, form, host, rounding, some_batch, some_cache

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


def tight(kind, want, size, total, reach, dim, blocks, small=31):
    """What scores in 32 bits, weights in two fp16 parts and one rounding to the type leave: each weight is off by 2^-22
    of itself, in the products and in the sum that divides them, or by 2^-small of its row's largest. blocks: the
    largest value of each column's block."""
    e = (dim // 32 * PARTS[kind] + 4) * 2.0 ** -22 * reach
    tol = size * (2 * e + 2.0 ** -20) + np.abs(want) * 2.0 ** -21 + rounding(want, TYPES[kind])
    return tol + total * 2.0 ** -small + blocks * 2.0 ** -32


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,fmt", [(64, "fp8"), (64, "fp4"), (128, "fp8"), (128, "fp4"), (256, "fp8"), (256, "fp4")])
@pytest.mark.parametrize("new,lengths,heads,columns", [([1, 1, 1], [300, 17, 2100], 8, None),
                                                       ([3, 1], [700, 90], 6, 600),
                                                       ([100, 130], [300, 130], 20, 2000)])
def test_results_are_rounded_once(gpu, new, lengths, heads, columns, dim, fmt, kind):
    """Whatever the kernel: nothing but the result's type rounds to fewer than 22 bits."""
    pages = sum(-(-n // 16) for n in lengths) + 1
    cache, codes, scales = some_cache(gpu, pages, 16, 2, dim, fmt, 221, big=0.0)
    batch, plain, rows = some_batch(gpu, new, lengths, 16, pages, 222, columns=columns)
    assert (form(kind, rows, heads, cache, batch)[0] == CHUNK) == (columns == 2000 and dim < 256)
    q = dev(0.1 * W.normal((rows, heads, dim), 223, 1.0), gpu, TYPES[kind])
    want, size, total, reach = O.attention(host(q), codes, scales, fmt, plain)
    blocks = np.exp2(scales[1].max((0, 1, 2)) - 127.0).repeat(32) * (448 if fmt == "fp8" else 6)
    close("once", paged.attention(q, cache, batch), want, tight(kind, want, size, total, reach, dim, blocks))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,columns", FORMS)
@pytest.mark.parametrize("gap", [10.0, 17.0, 23.0])
@pytest.mark.parametrize("length", [250, 4100])
def test_many_small_weights_beside_a_large_one(gpu, length, gap, heads, columns, kind):
    """A first token that takes the scores but has no value, and others `gap` below it, all alike, so that what their
    weights lose does not cancel: 2^-37 of the first one's each."""
    cache, codes, scales = some_cache(gpu, 65, 64, 2, 64, "fp8", 231)
    batch, plain, rows = some_batch(gpu, [40], [length], 64, 65, 232, columns=columns)
    assert (form(kind, rows, heads, cache, batch)[0] == CHUNK) == bool(columns)
    codes[0], scales[0] = 0, 0
    codes[1] &= 0x7f  # values of one sign, so that their sum does not cancel either
    page, slot = O.place(plain, 0, 0, 65, 64)
    codes[0, page, :, slot, 0], scales[0, page, :, slot, 0], codes[1, page, :, slot] = 0x38, 127, 0
    cache = on(gpu, codes, scales, "fp8")
    q = torch.zeros((rows, heads, 64), device=gpu, dtype=TYPES[kind])
    q[:, :, 0] = gap
    want, size, total, reach = O.attention(host(q), codes, scales, "fp8", plain, scale=1.0)
    blocks = np.exp2(scales[1].max((0, 1, 2)) - 127.0).repeat(32) * 448
    # The values' own error comes with the weights of those that have one: `length` of size / total at most.
    blocks = blocks * np.minimum(1, length * size / np.maximum(total, 1e-30))
    tol = tight(kind, want, size, total, reach, 64, blocks, 37)
    close("small", paged.attention(q, cache, batch, scale=1.0), want, tol)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,columns", FORMS)
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 27, 2.0 ** 29, 2.0 ** 33, 2.0 ** 60])
def test_scores_far_from_zero(gpu, size, heads, columns, kind):
    """One key, or equal ones, whose scores are large numbers, of either sign: the values' mean."""
    cache, codes, scales = some_cache(gpu, 20, 16, 2, 64, "fp8", 241)
    codes[0], scales[0] = 0, 0
    codes[0, ..., 0], scales[0, ..., 0] = 0x38, 127  # keys of (1, 0, ...)
    batch, plain, rows = some_batch(gpu, [70, 3], [170, 90], 16, 20, 242, columns=columns)
    cache = on(gpu, codes, scales, "fp8")
    rng = np.random.default_rng(243)
    q = size * (1 + rng.random((rows, heads, 64))) * rng.choice((-1, 1), (rows, heads, 1))
    q = dev(q, gpu, TYPES[kind])
    for window in (1, 37, None):
        want, mean, total, _ = O.attention(host(q), codes, scales, "fp8", plain, window=window)
        tol = (mean + np.abs(want)) * 2.0 ** -20 + rounding(want, TYPES[kind])
        close(f"{size} {window}", paged.attention(q, cache, batch, window=window), want, tol + total * 2.0 ** -31)


@pytest.mark.parametrize("heads,columns", FORMS)
def test_queries_up_to_the_largest_number(gpu, heads, columns):
    """fp32 queries at the end of their range over keys as small as scale bytes make them."""
    for low in (3, 8):
        cache, codes, scales = some_cache(gpu, 20, 16, 2, 64, "fp8", 261)
        codes[0] = codes[0] & 0x8f | 0x30  # 2^-1 to 2^-0.1, both signs
        scales[0] = low
        batch, plain, rows = some_batch(gpu, [70, 3], [170, 90], 16, 20, 262, columns=columns)
        cache = on(gpu, codes, scales, "fp8")
        q = dev(W.normal((rows, heads, 64), 263, 1.0), gpu) * 2.0 ** (127 - low)
        q[:, :, ::7] = torch.finfo(torch.float32).max * 2.0 ** (3 - low)
        q[::2, :, 1::7] = -torch.finfo(torch.float32).max * 2.0 ** (3 - low)
        assert torch.isfinite(q).all()
        want, size, total, reach = O.attention(host(q), codes, scales, "fp8", plain)
        blocks = np.exp2(scales[1].max((0, 1, 2)) - 127.0).repeat(32) * 448
        close(f"{low}", paged.attention(q, cache, batch), want, tight("f32", want, size, total, reach, 64, blocks))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,columns", [(4, None), (4, 600), (40, 9000)])
@pytest.mark.parametrize("first,last", [(0, 1024), (700, 1500), (0, 33)])
def test_scores_below_every_number(gpu, first, last, heads, columns, kind):
    """Keys whose scores pass fp32 to minus infinity have no weight, also where waves or workgroups have no other."""
    cache, codes, scales = some_cache(gpu, 110, 16, 2, 64, "fp8", 251, big=0.0)
    batch, plain, rows = some_batch(gpu, [20], [1600], 16, 110, 252, columns=columns)
    codes[0] &= 0x7f
    for t in range(1600):
        page, slot = O.place(plain, 0, t, 110, 16)
        scales[0, page, :, slot] = 127 + 40 if first <= t < last else 127 - 106
    cache = on(gpu, codes, scales, "fp8")
    q = dev(-np.abs(W.normal((rows, heads, 64), 253, 1.0)) * 2.0 ** 100, gpu, TYPES[kind])
    for window in (None, 1200):
        want, size, total, _ = O.attention(host(q), codes, scales, "fp8", plain, window=window)
        assert np.isfinite(want).all()
        # The largest scale sum |q k| of the keys that count: 64 products of 4.5 * 448 * 2^-6, over 8.
        tol = tight(kind, want, size, total, np.float64(256.0), 64, 448 * np.exp2(scales[1].max() - 127.0))
        close(f"{window}", paged.attention(q, cache, batch, window=window), want, tol)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,columns", [(4, None), (4, 600), (40, 9000)])
def test_nothing_but_scores_of_minus_infinity_is_a_nan(gpu, heads, columns, kind):
    """0 / 0, whether or not a row's keys are shared; rows beside it are as they were, and one without keys is 0."""
    cache, codes, scales = some_cache(gpu, 110, 16, 2, 64, "fp8", 255, big=0.0)
    codes[0] = np.maximum(codes[0] & 0x7f, 8)  # keys above 0 (a bit set in 0x77 would make it 0x7f, the NaN of e4m3)
    cache = on(gpu, codes, scales, "fp8")
    batch, plain, rows = some_batch(gpu, [20, 3], [1600, 2], 16, 110, 256, columns=columns)
    q = dev(W.normal((rows, heads, 64), 257, 1.0), gpu, TYPES[kind])
    q[5, 1, 7] = q[20, 0, 0] = q[21, heads - 1, 3] = float("-inf")  # row 20 is before the second sequence's first token
    got = torch.isnan(paged.attention(q, cache, batch)).cpu().numpy()
    want = np.zeros(got.shape, bool)
    want[5, 1] = want[21, heads - 1] = True
    assert np.array_equal(got, want)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,columns", [(4, None), (4, 600), (20, 9000)])
def test_a_nan_in_a_query_is_its_rows_alone(gpu, heads, columns, dim, kind):
    cache, codes, scales = some_cache(gpu, 80, 16, 2, dim, "fp8", 271)
    batch, plain, rows = some_batch(gpu, [30, 1], [1100, 40], 16, 80, 272, columns=columns)
    q = dev(W.normal((rows, heads, dim), 273, 1.0), gpu, TYPES[kind])
    want, size, total, reach = O.attention(host(q), codes, scales, "fp8", plain)
    q[7, 1, 5], q[30, heads - 1, dim - 1] = float("nan"), float("nan")
    want[7, 1] = want[30, heads - 1] = float("nan")
    blocks = np.exp2(scales[1].max((0, 1, 2)) - 127.0).repeat(32) * 448
    close("nan", paged.attention(q, cache, batch), want, tight(kind, want, size, total, reach, dim, blocks))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_write_turns_by_angles_up_to_the_limit(gpu, layout):
    """Positions up to 2^31 - 1 and frequencies up to 2^20: the oracle's codes."""
    freqs = [2.0 ** 20, -2.0 ** 20 + 0.5, 1e6 / 3, 2.0 ** 17 + 0.1, 2.0 ** 16 - 0.7, 777.7, 1.0, np.pi / 2, 1e-3]
    plan = paged.Rotary(torch.tensor(freqs, dtype=torch.float64, device=gpu), layout)
    page = 65536
    for length in (2 ** 31 - 1, 2 ** 30 + 12345, 2 ** 28 + 7):
        column = (length - 1) // page
        table = np.full((1, column + 1), -1, np.int32)
        table[0, column] = 0
        cache = paged.Cache.empty(1, page, 1, 64, "fp8", gpu)
        rows = 3000
        batch = paged.Batch(*(torch.from_numpy(a.copy()).to(gpu) for a in (
            np.array([0, rows], np.int32), np.array([length], np.int32), table)))
        k = dev(W.normal((rows, 1, 64), 281, 1.0), gpu)
        cache.write(k, k, batch, plan)
        at = np.arange(length - rows, length)
        here = at // page == column
        want, scales = OM.encode(O.rotate(host(k), at, freqs, layout).reshape(rows, 64)[here], "fp8")
        slots = torch.from_numpy(at[here] % page).to(gpu)
        assert np.array_equal(cache.scales[0, 0, 0, slots].cpu().numpy(), scales[:, :2])
        assert np.array_equal(cache.codes[0, 0, 0, slots].cpu().numpy(), want[:, :64])
