"""The paged operators on the GPU against the 64-bit oracle.

Rotary: cosine and sine to 2^-22 of their largest value (angle reduced in 64 bits, a few roundings of 2^-24 each), two
products and their sum (2^-24 each): within (|x| + |y|) m 2^-21 and the result's type. Written codes are rounded once
from 64 bits: the oracle's bytes.

Attention, with A = sum_j w_j |v_j| of a row: scores are sums of exact products, D / 32 instructions a part of q, each
of which adds at most one step (2^-23) of the largest of its terms twice; three parts hold 24 bits of q. With R the
largest scale sum |q k|, a score is within e = (D / 32 * parts + 4) 2^-22 R, and so the result within 2 e A.
Exponentials are good to 2^-21, weights to half a step of fp16 (fp32 results: 2^-21), in the products and in the sum
that divides them: 2^-11 (A + |o|). Each weight that is less than fp16 holds is off by 2^-25 where the largest is 2^6
to 2^15, so by 2^-31 of it: 2^-31 sum_j |v_j| in all. Values are off by 2^-25 where the largest of their block is 2^11
or more, less than 2^-32 of it. Then the result's type: half its eps, and below its normal values, where its steps no
longer shrink, half of their step (fp16: 2^-25).
"""
import numpy as np
import pytest
import torch

from ancha_amd import _native, fused, mx, paged
from ancha_amd import workload as W
from oracle import mx as OM
from oracle import paged as O

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PARTS = {"f32": 3, "f16": 2, "bf16": 1}


def dev(a, gpu, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(gpu).to(dtype)


def host(t):
    return t.detach().cpu().double().numpy()


def ints(values, gpu, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=gpu)


def rounding(want, dtype):
    """How far rounding to the type may be off: half a step, which is least_normal * eps below the normal values."""
    ends = torch.finfo(dtype)
    return np.maximum(np.abs(want), ends.smallest_normal) * ends.eps / 2


def close(name, got, want, tol):
    got = host(got)
    assert got.shape == want.shape, f"{name}: shape {got.shape}, expected {want.shape}"
    other = np.argwhere(np.isnan(got) != np.isnan(want))
    assert not len(other), f"{name}: NaN in {len(other)} other places, the first {other[0]}"
    with np.errstate(invalid="ignore"):
        off = np.nan_to_num(np.abs(got - want), nan=0.0) / np.nan_to_num(np.broadcast_to(tol, want.shape), nan=1.0)
    worst = off.max(initial=0.0)
    assert worst <= 1, f"{name}: {worst:.3g} of the tolerance at {np.unravel_index(off.argmax(), off.shape)}"


# ---- rotary


def rotary_tolerance(x, plan, want, dtype):
    n = plan.width // 2
    size = np.abs(x).copy()
    first = slice(0, n) if plan.layout == "half" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if plan.layout == "half" else slice(1, 2 * n, 2)
    size[..., first] = size[..., second] = size[..., first] + size[..., second]
    size[..., 2 * n:] = 0
    return size * plan.magnitude * 2.0 ** -21 + rounding(want, dtype)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,dim,width", [(1, 1, 2, 2), (3, 5, 6, 4), (1, 40, 128, 128), (17, 3, 96, 48),
                                                  (5, 2, 256, 100), (700, 2, 64, 64), (2, 1, 515, 514), (9, 3, 80, 22),
                                                  (2, 1, 2050, 2048)])
def test_rotary(gpu, rows, heads, dim, width, layout, kind):
    dtype = TYPES[kind]
    x = dev(W.normal((rows, heads, dim), 3, 1.0), gpu, dtype)
    freqs, magnitude = paged.frequencies(width, 10000.0, "yarn", 4.0, 2048)
    plan = paged.rotary_plan(width, 10000.0, layout, "yarn", 4.0, 2048, device=gpu)
    assert plan.magnitude == magnitude and plan.freqs.tolist() == freqs and plan.width == width
    at = (np.arange(rows) * 977) % 200_003
    want = O.rotate(host(x), at, freqs, layout, magnitude)
    tol = rotary_tolerance(host(x), plan, want, dtype)
    for ints_of in (torch.int32, torch.int64):
        close(f"rotary {ints_of}", paged.rotary(x, ints(at.tolist(), gpu, ints_of), plan), want, tol)


def test_rotary_far_and_negative_positions(gpu):
    x = dev(W.normal((6, 2, 64), 5, 1.0), gpu)
    plan = paged.rotary_plan(64, device=gpu)
    at = [-3, -200_000, 0, 2_000_000, 2 ** 31 + 5, 2 ** 40 + 7]
    want = O.rotate(host(x), at, plan.freqs.tolist())
    # The angle itself is rounded to 64 bits: half a step of it, 2^-53 |angle|, on either side.
    tol = rotary_tolerance(host(x), plan, want, x.dtype) + 4 * 2.0 ** -53 * np.abs(np.array(at, float))[:, None, None]
    close("far", paged.rotary(x, ints(at, gpu, torch.int64), plan), want, tol)


@pytest.mark.parametrize("kind", list(TYPES))
def test_rotary_layouts_and_batches(gpu, kind):
    dtype = TYPES[kind]
    base = dev(W.normal((11, 9, 131), 6, 1.0), gpu, dtype)
    plan = paged.rotary_plan(64, layout="interleaved", device=gpu)
    at = np.arange(11) * 5
    for name, x in (("columns", base[:, :, 1:97]), ("heads", base[:, 2:7, 3:]), ("rows", base[::2]),
                    ("swapped", base.transpose(0, 1)[:9]), ("strided", base[:, :, ::2]),
                    ("broadcast", base[:1].expand(11, 9, 131))):
        want = O.rotate(host(x), at[:x.shape[0]], plan.freqs.tolist(), "interleaved")
        got = paged.rotary(x, ints(at[:x.shape[0]].tolist(), gpu), plan)
        assert got.is_contiguous()
        close(name, got, want, rotary_tolerance(host(x), plan, want, dtype))
    # Three sequences, the second without rows, rows of none on both sides; the third has fewer tokens than rows.
    batch = paged.Batch(ints([2, 5, 5, 9], gpu), ints([40, 7, 3], gpu), ints([[0], [0], [0]], gpu))
    where = np.array([0, 0, 37, 38, 39, -1, 0, 1, 2, 0, 0])
    want = O.rotate(host(base), where, plan.freqs.tolist(), "interleaved")
    want[[0, 1, 9, 10]] = 0
    close("batch", paged.rotary(base, batch, plan), want, rotary_tolerance(host(base), plan, want, dtype))
    for shape in ((0, 3, 64), (4, 0, 64)):
        assert paged.rotary(torch.zeros(shape, device=gpu), ints([0] * shape[0], gpu), plan).shape == shape


# ---- cache


def some_cache(gpu, pages, page, heads, dim, fmt, seed, big=4.0):
    """A cache full of tokens: (paged.Cache, codes, scales) with blocks of different sizes."""
    rng = np.random.default_rng(seed)
    x = W.normal((2 * pages * heads * page, dim), seed, 1.0)
    x = x * np.exp2(rng.integers(-3, 4, (1, dim // 32)).repeat(32, 1)) * (1 + big * (rng.random(dim) < 0.05))
    codes, scales = OM.encode(x.astype(np.float32), fmt)
    size = dim if fmt == "fp8" else dim // 2
    codes = np.ascontiguousarray(codes[:, :size]).reshape(2, pages, heads, page, size)
    scales = np.ascontiguousarray(scales[:, :dim // 32]).reshape(2, pages, heads, page, dim // 32)
    cache = paged.Cache(torch.from_numpy(codes.copy()).to(gpu), torch.from_numpy(scales.copy()).to(gpu), fmt)
    return cache, codes, scales


def some_batch(gpu, new, lengths, page, pages, seed, columns=None, pad=0, first=0):
    """(paged.Batch, the oracle's, rows): each sequence its own pages in any order, -1 behind them."""
    rng = np.random.default_rng(seed)
    per = [-(-max(n, 0) // page) for n in lengths]
    order = rng.permutation(pages)
    assert sum(per) <= pages
    table = np.full((len(new), columns or max(per + [1])), -1, np.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    starts = (first + np.concatenate(([0], np.cumsum(new)))).astype(np.int32)
    lengths = np.array(lengths, np.int32)
    batch = paged.Batch(*(torch.from_numpy(a.copy()).to(gpu) for a in (starts, lengths, table)))
    return batch, (starts, lengths, table), int(starts[-1]) + pad


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("heads,dim,page,width,layout", [(1, 64, 16, 0, "half"), (3, 64, 32, 64, "half"),
                                                         (2, 128, 16, 128, "interleaved"), (8, 128, 64, 20, "half"),
                                                         (5, 256, 128, 256, "half"), (3, 128, 16, 6, "interleaved")])
def test_write_and_read(gpu, heads, dim, page, width, layout, fmt, kind):
    dtype = TYPES[kind]
    cache, codes, scales = some_cache(gpu, 24, page, heads, dim, fmt, 11)
    new, lengths = [1, 0, 33, 4, 2], [50, 20, 33, 2, 17]  # the fourth has rows before its first token
    batch, plain, rows = some_batch(gpu, new, lengths, page, 24, 12, pad=3, first=2)
    k, v = (dev(W.normal((rows, heads, dim), s, 1.0), gpu, dtype) for s in (13, 14))
    k[4, 0, :32] = 0
    plan, key = None, host(k)
    if width:
        plan = paged.rotary_plan(width, layout=layout, device=gpu)
        at = np.zeros(rows)
        for r, _, position in O.rows_of(plain, rows):
            at[r] = position
        key = O.rotate(host(k), at, plan.freqs.tolist(), layout)
    assert cache.write(k, v, batch, plan) is cache
    O.write(codes, scales, fmt, key, host(v), plain)
    assert np.array_equal(cache.scales.cpu().numpy(), scales)
    assert np.array_equal(cache.codes.cpu().numpy(), codes)
    for size in (1, 35, 60):
        got = cache.read(batch, size, dtype)
        for i in range(len(new)):
            want = O.sequence(codes, scales, fmt, plain, i, size)
            for which in (0, 1):
                assert torch.equal(got[which][i].cpu(), torch.from_numpy(want[which]).to(dtype)), (size, i, which)
    assert cache.read(batch, 0)[0].shape == (5, 0, heads, dim)


def test_write_turns_by_any_angle(gpu):
    """Angles within rounding of a right angle's multiples, small ones, and up to 2^28."""
    cache, codes, scales = some_cache(gpu, 4, 64, 2, 64, "fp8", 24)
    quarter = np.pi / 2
    freqs = [quarter, np.nextafter(quarter, 2), -quarter / 2, 1e-9, 0.0, 1.0, -3.7, 512.5, 1e6, 2.0 ** 20 - 0.3]
    plan = paged.Rotary(torch.tensor(freqs, dtype=torch.float64, device=gpu))
    batch, plain, rows = some_batch(gpu, [200], [230], 64, 4, 25)
    k = dev(W.normal((rows, 2, 64), 26, 1.0), gpu)
    cache.write(k, k, batch, plan)
    at = np.zeros(rows)
    for r, _, position in O.rows_of(plain, rows):
        at[r] = position
    O.write(codes, scales, "fp8", O.rotate(host(k), at, freqs), host(k), plain)
    assert np.array_equal(cache.scales.cpu().numpy(), scales)
    assert np.array_equal(cache.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_write_special_values_and_layouts(gpu, fmt):
    cache, codes, scales = some_cache(gpu, 4, 16, 2, 64, fmt, 21)
    packed = dev(W.normal((7, 6, 130), 22, 1.0), gpu)
    packed[0, 2, 70], packed[1, 3, 3], packed[2, 4, 65] = float("nan"), float("inf"), float("-inf")
    packed[3, 2] = 3e38
    packed[4, 4] = 2.0 ** -149
    batch, plain, _ = some_batch(gpu, [4, 3], [20, 3], 16, 4, 23)
    for k, v in ((packed[:, 2:4, :64], packed[:, 4:, 1:65]), (packed[:, 2:4, 65:129], packed[:, 4:, 2::2]),
                 (packed[:1, 2:4, :64].expand(7, 2, 64), packed[:, :1, :64].expand(7, 2, 64))):
        assert cache.write(k, v, batch) is cache
        O.write(codes, scales, fmt, host(k), host(v), plain)
        assert np.array_equal(cache.scales.cpu().numpy(), scales)
        assert np.array_equal(cache.codes.cpu().numpy(), codes)
    empty = torch.zeros((0, 2, 64), device=gpu)
    assert cache.write(empty, empty, paged.Batch(ints([0], gpu), ints([], gpu), torch.zeros((0, 3), dtype=torch.int32,
                                                                                           device=gpu))) is cache


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("layout,width", [("half", 64), ("half", 40), ("interleaved", 64), ("interleaved", 36)])
def test_write_turns_special_values(gpu, layout, width, fmt):
    """NaN, infinities and sums of 2^128 or more in a turned key make their blocks NaN, no others."""
    cache, codes, scales = some_cache(gpu, 4, 16, 3, 64, fmt, 27)
    batch, plain, rows = some_batch(gpu, [9], [21], 16, 4, 28)
    plan = paged.rotary_plan(width, layout=layout, device=gpu)
    k = dev(W.normal((rows, 3, 64), 29, 1.0), gpu)
    k[0, 0, 0], k[1, 1, 33], k[2, 2, 5], k[3, 0, 63] = float("nan"), float("inf"), float("-inf"), float("inf")
    k[4, 1] = 3.3e38
    k[5, 2] *= 2.0 ** -130
    k[6, 0] = 0.0
    at = np.zeros(rows)
    for r, _, position in O.rows_of(plain, rows):
        at[r] = position
    with np.errstate(invalid="ignore"):
        turned = O.rotate(host(k), at, plan.freqs.tolist(), layout)
    turned[np.abs(turned) >= 2.0 ** 128] = np.inf
    assert np.isinf(turned[4, 1]).any() and np.isfinite(turned[4, 1]).any()
    cache.write(k, -k.flip(2), batch, plan)
    O.write(codes, scales, fmt, turned, host(-k.flip(2)), plain)
    assert np.array_equal(cache.scales.cpu().numpy(), scales)
    assert np.array_equal(cache.codes.cpu().numpy(), codes)


def test_pages_that_are_not_there(gpu):
    """Numbers outside the cache, columns behind the table and places below 0: not written, read as zeros, not seen."""
    cache, codes, scales = some_cache(gpu, 6, 16, 2, 64, "fp8", 31)
    table = np.array([[2, -1, 5, 6], [2 ** 31 - 1, 1, -2 ** 31, 0]], np.int32)
    plain = (np.array([0, 70, 80], np.int32), np.array([70, 64], np.int32), table)
    batch = paged.Batch(*(torch.from_numpy(a.copy()).to(gpu) for a in plain))
    k, v = dev(W.normal((80, 2, 64), 32, 1.0), gpu), dev(W.normal((80, 2, 64), 33, 1.0), gpu)
    assert cache.write(k, v, batch) is cache
    O.write(codes, scales, "fp8", host(k), host(v), plain)
    assert np.array_equal(cache.codes.cpu().numpy(), codes)
    got = cache.read(batch, 100, torch.float32)
    for i in (0, 1):
        want = O.sequence(codes, scales, "fp8", plain, i, 100)
        for which in (0, 1):
            assert np.array_equal(host(got[which][i]), want[which])
    for causal, window in ((True, None), (False, None), (True, 5)):
        check_attention(gpu, "f32", 4, cache, codes, scales, batch, plain, 80, 34, causal=causal, window=window)


# ---- attention


def check_attention(gpu, kind, heads, cache, codes, scales, batch, plain, rows, seed, q=None, **how):
    dtype = TYPES[kind]
    if q is None:
        q = dev(2 * W.normal((rows, heads, cache.dim), seed, 1.0), gpu, dtype)
    want, size, total, reach = O.attention(host(q), codes, scales, cache.format, plain, **how)
    got = paged.attention(q, cache, batch, **how)
    assert got.dtype == dtype and got.is_contiguous()
    e = (cache.dim // 32 * PARTS[kind] + 4) * 2.0 ** -22 * reach
    weights = 2.0 ** -21 if kind == "f32" else torch.finfo(torch.float16).eps / 2
    held = np.exp2(np.where(scales == 255, 0, scales).max() - 127.0) * (448 if cache.format == "fp8" else 6)
    tol = size * (2 * e + weights + 2.0 ** -21) + np.abs(want) * weights + rounding(want, dtype) + held * 2.0 ** -32
    tol = tol + total * 2.0 ** -31
    close(f"attention {kind} {how}", got, want, tol)
    return got


SHAPES = [  # new tokens, lengths, heads, cache heads, page
    ([1], [1], 1, 1, 16),
    ([1, 1, 1], [16, 17, 300], 8, 2, 16),
    ([1] * 5, [33, 1, 0, 64, 127], 15, 3, 32),
    ([7, 0, 40, 1], [7, 50, 90, 70], 4, 4, 16),
    ([3, 21], [500, 21], 12, 1, 64),
    ([5, 2], [3, 1], 5, 5, 16),  # more rows than tokens: the first ones see nothing
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,fmt", [(64, "fp8"), (64, "fp4"), (128, "fp8"), (128, "fp4"), (256, "fp8"), (256, "fp4")])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(gpu, shape, dim, fmt, kind):
    new, lengths, heads, kv, page = SHAPES[shape]
    pages = sum(-(-n // page) for n in lengths) + 2
    cache, codes, scales = some_cache(gpu, pages, page, kv, dim, fmt, 41)
    batch, plain, rows = some_batch(gpu, new, lengths, page, pages, 42, pad=shape % 2 * 3, first=shape % 3)
    for how in ({}, {"causal": False}, {"window": 9}, {"causal": False, "window": 2, "scale": 0.3}):
        check_attention(gpu, kind, heads, cache, codes, scales, batch, plain, rows, 43, **how)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_attention_over_a_long_cache(gpu, fmt, kind):
    """Few rows and many keys: shared out over workgroups whose parts are joined."""
    cache, codes, scales = some_cache(gpu, 200, 16, 2, 64, fmt, 51)
    batch, plain, rows = some_batch(gpu, [1, 2, 3], [2500, 400, 5], 16, 200, 52, columns=300, pad=1)
    for how in ({}, {"window": 700}, {"causal": False}):
        check_attention(gpu, kind, 8, cache, codes, scales, batch, plain, rows, 53, **how)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_of_many_sequences(gpu, kind):
    rng = np.random.default_rng(61)
    new, lengths = rng.integers(0, 3, 150).tolist(), rng.integers(0, 60, 150).tolist()
    cache, codes, scales = some_cache(gpu, 700, 16, 1, 64, "fp8", 62)
    batch, plain, rows = some_batch(gpu, new, lengths, 16, 700, 63, pad=5)
    check_attention(gpu, kind, 6, cache, codes, scales, batch, plain, rows, 64)


TILES4, TILES8, CHUNK = 0, 1, 2


def form(kind, rows, heads, cache, batch):
    """(kernel, workgroups that may share a tile's keys) of a call."""
    got = _native.lib().ancha_amd_paged_form(list(TYPES).index(kind), rows, heads, cache.heads, cache.dim, len(batch),
                                             batch.table.shape[1] * cache.page)
    return got % 3, got // 3


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,fmt", [(64, "fp8"), (64, "fp4"), (128, "fp8"), (128, "fp4"), (256, "fp8")])
@pytest.mark.parametrize("new,lengths,heads,kv,page,columns", [
    ([257, 130, 1], [257, 411, 300], 4, 2, 32, 44),       # tiles of 16 rows
    ([257, 130, 80], [257, 411, 300], 4, 2, 32, 600),     # room for long sequences: the chunk kernel, shared keys
    ([64, 100], [900, 100], 16, 2, 16, 1200),             # shared by several, the last part short
    ([100, 0, 37, 90], [64, 50, 1100, 90], 21, 3, 64, 500),  # rows without keys, sevens of heads
])
def test_attention_of_chunks(gpu, new, lengths, heads, kv, page, columns, dim, fmt, kind):
    pages = sum(-(-n // page) for n in lengths) + 1
    cache, codes, scales = some_cache(gpu, pages, page, kv, dim, fmt, 71)
    batch, plain, rows = some_batch(gpu, new, lengths, page, pages, 72, columns=columns, pad=2, first=1)
    kernel, shares = form(kind, rows, heads, cache, batch)
    assert kernel == (CHUNK if dim < 256 and columns > 100 else TILES8 if dim < 256 else TILES4)
    assert shares > 1 or dim == 256
    for how in ({}, {"window": 100}, {"causal": False}):
        check_attention(gpu, kind, heads, cache, codes, scales, batch, plain, rows, 73, **how)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_of_whole_prompts(gpu, kind):
    """As many tiles as run at once: nobody shares their keys."""
    cache, codes, scales = some_cache(gpu, 34, 16, 32, 64, "fp8", 75)
    batch, plain, rows = some_batch(gpu, [270, 200], [270, 210], 16, 34, 76, columns=1000)
    assert form(kind, rows, 128, cache, batch) == (CHUNK, 1)
    q = dev(W.normal((rows, 128, 64), 77, 1.0), gpu, TYPES[kind])
    few = slice(0, 128, 29)  # the oracle on some heads: 0, 29, .. read heads 0, 7, .. of the cache
    heads = [h // 4 for h in range(0, 128, 29)]
    got = paged.attention(q, cache, batch)[:, few]
    part = np.ascontiguousarray(codes[:, :, heads]), np.ascontiguousarray(scales[:, :, heads])
    want, size, total, reach = O.attention(host(q[:, few]), *part, "fp8", plain)
    e = (2 * PARTS[kind] + 4) * 2.0 ** -22 * reach
    tol = size * (2 * e + 2.0 ** -11 + 2.0 ** -21) + np.abs(want) * 2.0 ** -11 + rounding(want, TYPES[kind])
    close("prompts", got, want, tol + total * 2.0 ** -31 + np.exp2(scales.max() - 127.0) * 448 * 2.0 ** -32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim,fmt", [(64, "fp4"), (128, "fp8")])
def test_attention_of_a_thousand_tiles(gpu, dim, fmt, kind):
    rng = np.random.default_rng(65)
    lengths = rng.integers(0, 40, 140).tolist()
    cache, codes, scales = some_cache(gpu, 420, 16, 8, dim, fmt, 66)
    batch, plain, rows = some_batch(gpu, [1] * 140, lengths, 16, 420, 67)
    assert form(kind, rows, 8, cache, batch)[0] == TILES4
    check_attention(gpu, kind, 8, cache, codes, scales, batch, plain, rows, 68)


def test_attention_what_was_not_written_is_not_seen(gpu):
    """NaN codes and scales behind the sequences' ends, before the window and in pages of nobody."""
    for dim, fmt, new, columns in ((64, "fp8", 1, None), (128, "fp4", 1, None), (256, "fp8", 1, None),
                                   (64, "fp8", 30, 9000), (128, "fp4", 30, 9000)):
        cache, codes, scales = some_cache(gpu, 12, 16, 2, dim, fmt, 81)
        batch, plain, rows = some_batch(gpu, [new, 20], [37, 50], 16, 12, 82, columns=columns)
        heads = 2 if columns is None else 20
        assert form("bf16", rows, heads, cache, batch)[0] == (CHUNK if columns else TILES4 if dim > 128 else TILES8)
        used = np.zeros((12, 16), bool)
        for i, length in enumerate(plain[1]):
            for t in range(length):
                used[O.place(plain, i, t, 12, 16)] = True
        codes.transpose(1, 3, 0, 2, 4)[~used], scales.transpose(1, 3, 0, 2, 4)[~used] = 0x7f, 255
        cache = paged.Cache(torch.from_numpy(codes.copy()).to(gpu), torch.from_numpy(scales.copy()).to(gpu), fmt)
        for how in ({}, {"window": 6}, {"causal": False}):
            check_attention(gpu, "bf16", heads, cache, codes, scales, batch, plain, rows, 83, **how)


@pytest.mark.parametrize("dim,fmt,heads,columns", [
    (64, "fp8", 4, None), (64, "fp4", 4, None), (128, "fp8", 4, None), (128, "fp4", 4, None), (256, "fp8", 4, None),
    (256, "fp4", 4, None), (64, "fp8", 20, 4000), (64, "fp4", 20, 4000), (128, "fp8", 20, 4000),
    (128, "fp4", 20, 4000)])
def test_attention_a_nan_reaches_the_rows_that_see_it(gpu, dim, fmt, heads, columns):
    cache, codes, scales = some_cache(gpu, 12, 16, 2, dim, fmt, 91)
    batch, plain, rows = some_batch(gpu, [40, 1], [70, 90], 16, 12, 92, columns=columns)
    assert (form("bf16", rows, heads, cache, batch)[0] == CHUNK) == bool(columns)
    page, slot = O.place(plain, 0, 45, 12, 16)  # seen by the rows from position 45 on
    for which, head, block in ((0, 0, 1), (1, 1, 0), (1, 1, dim // 32 - 1)):
        scales[which, page, head, slot, block], codes[which, page, head, slot].reshape(dim // 32, -1)[block] = 255, 0
    page, slot = O.place(plain, 1, 3, 12, 16)
    scales[1, page, 0, slot, 1], codes[1, page, 0, slot].reshape(dim // 32, -1)[1] = 255, 0
    cache = paged.Cache(torch.from_numpy(codes.copy()).to(gpu), torch.from_numpy(scales.copy()).to(gpu), fmt)
    for kind in TYPES:
        for how in ({}, {"window": 10}, {"causal": False}):
            got = check_attention(gpu, kind, heads, cache, codes, scales, batch, plain, rows, 93, **how)
            assert torch.isnan(got).any() and not torch.isnan(got).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,columns", [(2, None), (12, 9000)])
def test_attention_blocks_and_scores_of_any_size(gpu, heads, columns, kind):
    """Values whose blocks grow by powers of two along the sequence, up and down, and scores that leave one key all."""
    for fmt, dim in (("fp8", 128), ("fp4", 64)):
        cache, codes, scales = some_cache(gpu, 20, 16, 1, dim, fmt, 101)
        batch, plain, rows = some_batch(gpu, [3, 50], [150, 160], 16, 20, 102, columns=columns)
        assert (form(kind, rows, heads, cache, batch)[0] == CHUNK) == bool(columns)
        for i in (0, 1):
            for t in range(int(plain[1][i])):
                page, slot = O.place(plain, i, t, 20, 16)
                scales[1, page, :, slot, 0] = 60 + t if i == 0 else 240 - t
                scales[1, page, :, slot, 1] = 100 + (t * 7919) % 40
        cache = paged.Cache(torch.from_numpy(codes.copy()).to(gpu), torch.from_numpy(scales.copy()).to(gpu), fmt)
        for sharp in (0.01, 1.0, 300.0):
            q = dev(sharp * W.normal((rows, heads, dim), 103, 1.0), gpu, TYPES[kind])
            want, size, total, reach = O.attention(host(q), codes, scales, fmt, plain)
            e = (dim // 32 * PARTS[kind] + 4) * 2.0 ** -22 * reach
            # A value is off by 2^-32 of the largest of its own block of columns, however large the others are.
            weights = 2.0 ** -21 if kind == "f32" else 2.0 ** -11
            tol = size * (2 * np.minimum(e, 1) + weights + 2.0 ** -21) + np.abs(want) * weights
            tol = tol + rounding(want, TYPES[kind])
            blocks = np.exp2(scales[1].max((0, 1, 2)) - 127.0).repeat(32) * (448 if fmt == "fp8" else 6)
            got = paged.attention(q, cache, batch)
            tol = tol + total * 2.0 ** -31 + blocks * 2.0 ** -32
            if kind == "f16":  # infinite from 65520 on, which what is within the tolerance of it may pass or not
                there = np.isinf(host(got)) & (np.sign(host(got)) * want + tol >= 65520)
                want, got = np.where(there, 0, want), got.masked_fill(torch.from_numpy(there).to(gpu), 0)
            close(f"{fmt} {sharp}", got, want, tol)


def test_attention_layouts(gpu):
    cache, codes, scales = some_cache(gpu, 8, 16, 2, 64, "fp8", 111)
    batch, plain, rows = some_batch(gpu, [3, 6], [30, 45], 16, 8, 112)
    base = dev(W.normal((18, 9, 140), 113, 1.0), gpu, torch.bfloat16)
    for name, q in (("columns", base[:9, :4, 1:65]), ("rows", base[::2, 1:7, 70:134]),
                    ("strided", base[:9, :2, ::2][..., :64]), ("swapped", base[:4].transpose(0, 1)[:, :, :64]),
                    ("broadcast", base[:1, :4, :64].expand(9, 4, 64))):
        check_attention(gpu, "bf16", q.shape[1], cache, codes, scales, batch, plain, rows, 0, q=q)


def test_attention_infinite_queries(gpu):
    """A row whose scores are all minus infinity, or one of them plus infinity, is NaN; its neighbours are not."""
    cache, codes, scales = some_cache(gpu, 4, 16, 1, 64, "fp8", 121)
    codes[0] = 0x38  # keys of ones
    scales[0] = 127
    cache = paged.Cache(torch.from_numpy(codes.copy()).to(gpu), torch.from_numpy(scales.copy()).to(gpu), "fp8")
    batch, plain, rows = some_batch(gpu, [4], [40], 16, 4, 122)
    q = torch.ones((4, 2, 64), device=gpu)
    q[1, 0, 3], q[2, 1, 5] = float("-inf"), float("inf")
    got = paged.attention(q, cache, batch)
    nan = torch.isnan(got).all(2).cpu()
    assert nan.tolist() == [[False, False], [True, False], [False, True], [False, False]]
    assert torch.isnan(got).any(2).cpu().equal(nan)


@pytest.mark.parametrize("rows", [1, 9, 40, 170])
def test_a_batch_of_more_rows_than_there_are(gpu, rows):
    """The first rows of a batch's: each at the position that the batch gives it, in a write, a turn and attention."""
    cache, codes, scales = some_cache(gpu, 40, 16, 2, 64, "fp8", 71)
    batch, plain, _ = some_batch(gpu, [8, 0, 30, 200], [100, 5, 30, 210], 16, 40, 72)
    plan = paged.rotary_plan(64, device=gpu)
    k, v = dev(W.normal((rows, 2, 64), 73, 1.0), gpu), dev(W.normal((rows, 2, 64), 74, 1.0), gpu)
    at = np.zeros(rows)
    for r, _, position in O.rows_of(plain, rows):
        at[r] = position
    turned = O.rotate(host(k), at, plan.freqs.tolist())
    cache.write(k, v, batch, plan)
    O.write(codes, scales, "fp8", turned, host(v), plain)
    assert np.array_equal(cache.codes.cpu().numpy(), codes) and np.array_equal(cache.scales.cpu().numpy(), scales)
    close("rotary", paged.rotary(k, batch, plan), turned, rotary_tolerance(host(k), plan, turned, torch.float32))
    for causal, window in ((True, None), (False, None), (True, 7), (True, 2 ** 70)):
        check_attention(gpu, "bf16", 8, cache, codes, scales, batch, plain, rows, 75, causal=causal, window=window)


def test_attention_of_nothing(gpu):
    cache, _, _ = some_cache(gpu, 4, 16, 2, 64, "fp8", 131)
    none = paged.Batch(ints([0], gpu), ints([], gpu), torch.zeros((0, 3), dtype=torch.int32, device=gpu))
    bare = paged.Batch(ints([0, 4], gpu), ints([9], gpu), torch.zeros((1, 0), dtype=torch.int32, device=gpu))
    q = torch.ones((5, 4, 64), device=gpu)
    for batch in (none, bare):
        got = paged.attention(q, cache, batch)
        assert got.shape == q.shape and not got.any()
    assert paged.attention(q[:0], cache, none).shape == (0, 4, 64)
    k, v = cache.read(bare, 7)
    assert k.shape == (1, 7, 2, 64) and not k.any() and not v.any()


def test_pages_far_apart(gpu):
    """Codes behind 2^32 bytes: the last pages of a cache of 9 GiB."""
    pages = (1 << 32) // (8 * 64 * 128) + 700
    cache = paged.Cache.empty(pages, 64, 8, 128, "fp8", gpu)
    table = np.array([[pages - 1, 0, pages - 300]], np.int32)
    plain = (np.array([0, 150], np.int32), np.array([150], np.int32), table)
    batch = paged.Batch(*(torch.from_numpy(a).to(gpu) for a in plain))
    k, v = (dev(W.normal((150, 8, 128), s, 1.0), gpu, torch.bfloat16) for s in (141, 142))
    cache.write(k, v, batch)
    codes, scales = np.zeros((2, 3, 8, 64, 128), np.uint8), np.zeros((2, 3, 8, 64, 4), np.uint8)
    near = (plain[0], plain[1], np.array([[0, 1, 2]], np.int32))
    O.write(codes, scales, "fp8", host(k), host(v), near)
    at = torch.from_numpy(table[0].astype(np.int64)).to(gpu)
    assert np.array_equal(cache.codes[:, at].cpu().numpy(), codes)
    assert np.array_equal(cache.scales[:, at].cpu().numpy(), scales)
    got = cache.read(batch, 150, torch.float32)
    want = O.sequence(codes, scales, "fp8", near, 0, 150)
    assert np.array_equal(host(got[1][0]), want[1])
    q = dev(W.normal((150, 8, 128), 143, 1.0), gpu, torch.bfloat16)
    check_attention(gpu, "bf16", 8, cache, codes, scales, batch, near, 150, 0, q=q)
    del cache, got
    torch.cuda.empty_cache()


def test_wrappers_check_shapes_types_and_devices(gpu):
    cache, _, _ = some_cache(gpu, 4, 16, 2, 64, "fp8", 145)
    batch, _, rows = some_batch(gpu, [2, 1], [20, 9], 16, 4, 146)
    plan, wide = paged.rotary_plan(64, device=gpu), paged.rotary_plan(66, device=gpu)
    x, at = torch.ones((rows, 2, 64), device=gpu), ints([0] * rows, gpu)
    for text, call in (
            ("rows, heads, dim", lambda: paged.rotary(x[0], at, plan)),
            ("float32, float16 or bfloat16", lambda: paged.rotary(x.double(), at, plan)),
            ("turns 66", lambda: paged.rotary(x, at, wide)),
            ("shape", lambda: paged.rotary(x, at[:2], plan)),
            ("int32 or int64", lambda: paged.rotary(x, at.float(), plan)),
            ("must be on", lambda: paged.rotary(x, at.cpu(), plan)),
            ("paged.Rotary", lambda: paged.rotary(x, at, None)),
            ("turns 66", lambda: cache.write(x, x, batch, wide)),
            (r"\[rows, 2, 64\]", lambda: cache.write(x[:, :1], x[:, :1], batch)),
            ("shape", lambda: cache.write(x, x[:2], batch)),
            ("torch.float32", lambda: cache.write(x, x.half(), batch)),
            ("paged.Batch", lambda: cache.write(x, x, at)),
            ("size", lambda: cache.read(batch, -1)),
            ("dtype", lambda: cache.read(batch, 3, torch.int8)),
            ("multiple of 2 heads", lambda: paged.attention(x[:, :1], cache, batch)),
            ("64 columns", lambda: paged.attention(x[:, :, :32], cache, batch)),
            ("window", lambda: paged.attention(x, cache, batch, window=0)),
            ("scale", lambda: paged.attention(x, cache, batch, scale=0.0)),
            ("paged.Cache", lambda: paged.attention(x, batch, batch)),
            ("int32", lambda: paged.Batch(batch.starts.long(), batch.lengths, batch.table)),
            ("shape", lambda: paged.Batch(batch.starts[:2], batch.lengths, batch.table)),
            ("shape", lambda: paged.Batch(batch.starts, batch.lengths, batch.table[:1])),
            ("contiguous", lambda: paged.Batch(batch.starts, batch.lengths, batch.table.t().contiguous().t())),
            ("contiguous", lambda: paged.Cache(cache.codes.transpose(0, 2), cache.scales, "fp8")),
            ("shape", lambda: paged.Cache(cache.codes, cache.scales[:, :3].contiguous(), "fp8")),
            ("bytes of", lambda: paged.Cache(cache.codes[..., :32].contiguous(), cache.scales, "fp8")),
            ("power of two", lambda: paged.Cache.empty(4, 24, 2, 64, "fp8", gpu)),
            ("at least one page", lambda: paged.Cache.empty(0, 16, 2, 64, "fp8", gpu)),
            ("magnitude", lambda: paged.Rotary(plan.freqs, "half", 0.0)),
            ("empty", lambda: paged.Rotary(plan.freqs[:0]))):
        with pytest.raises(ValueError, match=text):
            call()


# ---- together


def layer(x, w_qkv, w_out, heads, kv, plan, cache, batch):
    """A layer's attention on microscaled weights, as a served model runs it."""
    dim = cache.dim
    y, stream = mx.add_unit_norm(x, torch.zeros_like(x), None, 1e-6)
    qkv = mx.linear(y, w_qkv, dtype=torch.bfloat16).view(-1, heads + 2 * kv, dim)
    q, k, v = qkv.split((heads, kv, kv), 1)
    assert cache.write(k, v, batch, plan) is cache
    out = paged.attention(paged.rotary(q, batch, plan), cache, batch)
    return mx.linear(mx.quantize(out.flatten(1), "fp8"), w_out, fused.Epilogue(residual=stream),
                     dtype=torch.bfloat16), (q, k, v, out)


def test_a_layer_token_by_token(gpu):
    """A prompt and then tokens of two sequences through a layer: every step's operators against the oracle on the same
    projections, into one cache that the oracle keeps too."""
    heads, kv, dim, width = 6, 2, 64, 256
    w_qkv = mx.weight(dev(W.normal((width, (heads + 2 * kv) * dim), 151, width ** -0.5), gpu))
    w_out = mx.weight(dev(W.normal((heads * dim, width), 152, 0.05), gpu))
    plan = paged.rotary_plan(dim, 10000.0, "half", "ntk", 2.0, device=gpu)
    cache = paged.Cache.empty(9, 16, kv, dim, "fp8", gpu)
    codes, scales = np.zeros((2, 9, kv, 16, dim), np.uint8), np.zeros((2, 9, kv, 16, 2), np.uint8)
    table = np.array([[7, 2, 4, -1], [1, 0, 8, 3]], np.int32)
    grown = ([20, 37], [20, 37]), ([1, 1], [21, 38]), ([0, 5], [21, 43]), ([1, 1], [22, 44])
    for step, (new, lengths) in enumerate(grown):
        plain = (np.concatenate(([0], np.cumsum(new))).astype(np.int32), np.array(lengths, np.int32), table)
        batch = paged.Batch(*(torch.from_numpy(a).to(gpu) for a in plain))
        rows = sum(new)
        x = dev(W.normal((rows, width), 153 + step, 1.0), gpu, torch.bfloat16)
        out, (q, k, v, mixed) = layer(x, w_qkv, w_out, heads, kv, plan, cache, batch)
        assert out.shape == x.shape and torch.isfinite(out).all()
        at = [position for _, _, position in O.rows_of(plain, rows)]
        O.write(codes, scales, "fp8", O.rotate(host(k), at, plan.freqs.tolist()), host(v), plain)
        assert np.array_equal(cache.codes.cpu().numpy(), codes) and np.array_equal(cache.scales.cpu().numpy(), scales)
        turned = paged.rotary(q, batch, plan)
        want = check_attention(gpu, "bf16", heads, cache, codes, scales, batch, plain, rows, 0, q=turned)
        assert torch.equal(mixed, want)


def test_captured_steps_on_new_lengths(gpu):
    """A decoding step captured once and replayed while sequences grow: each replay equals the same call made eagerly,
    with other work and synchronisation between them, and two graphs run on their own streams."""
    heads, kv, dim = 8, 2, 128
    plan = paged.rotary_plan(dim, device=gpu)
    plain_k = dev(W.normal((40, 4, kv, dim), 161, 1.0), gpu, torch.bfloat16)
    plain_q = dev(W.normal((40, 4, heads, dim), 162, 1.0), gpu, torch.bfloat16)

    class Step:
        def __init__(self, seed):
            self.cache, _, _ = some_cache(gpu, 60, 16, kv, dim, "fp8", seed)
            self.batch, _, _ = some_batch(gpu, [1] * 4, [200, 3, 90, 160], 16, 60, seed, columns=20)
            self.q, self.k = torch.zeros_like(plain_q[0]), torch.zeros_like(plain_k[0])

        def run(self):
            self.cache.write(self.k, self.k, self.batch, plan)
            return paged.attention(paged.rotary(self.q, self.batch, plan), self.cache, self.batch)

        def set(self, i):
            self.q.copy_(plain_q[i])
            self.k.copy_(plain_k[i])
            self.batch.lengths.add_(1)
            if i == 2:
                self.batch.starts.copy_(ints([0, 0, 1, 3, 3], gpu))  # other rows than one each

    steps = [Step(163), Step(164)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for s in steps:
            s.run()
    torch.cuda.current_stream().wait_stream(side)
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in steps]
    for i in range(5):
        for s in steps:
            s.set(i)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for s, o in zip(steps, got):
            codes = s.cache.codes.clone()
            assert torch.equal(s.run(), o), f"replay {i}"
            assert torch.equal(s.cache.codes, codes)


def test_streams_and_repeats_give_the_same_bits(gpu):
    cache, _, _ = some_cache(gpu, 200, 16, 2, 128, "fp8", 171)
    batch, _, rows = some_batch(gpu, [1, 40], [1500, 900], 16, 200, 172, columns=100)
    q = dev(W.normal((rows, 8, 128), 173, 1.0), gpu, torch.bfloat16)
    want = paged.attention(q, cache, batch)
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            outs.append([paged.attention(q, cache, batch) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for some in outs for o in some)
