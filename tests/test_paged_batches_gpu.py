"""Batches of the paged operators that others do not reach: more than 64 sequences of several tiles, and values on the
device that keep no order, which no kernel may follow out of its tensors."""
import ctypes

import numpy as np
import pytest
import torch

from ancha_amd import _native, paged
from ancha_amd import workload as W
from oracle import paged as O
from tests.test_paged_gpu import CHUNK, TILES4, TILES8, TYPES, close, dev, form, host, ints, rotary_tolerance, \
    some_batch, some_cache
from tests.test_paged_numbers_gpu import tight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim,fmt", [(64, "fp8"), (128, "fp4")])
@pytest.mark.parametrize("columns", [None, 9000])
def test_tiles_behind_the_64th_sequence(gpu, dim, fmt, columns, kind):
    """150 sequences of up to 20 tiles of 16 rows, or three chunks, some without rows; rows of none around them."""
    rng = np.random.default_rng(301)
    most = 80 if dim == 64 else 160 if columns else 40
    new = rng.integers(most // 8, most + 1, 150)
    new[[0, 63, 64, 90, 128, 149]] = 0
    lengths = new + rng.integers(0, 30, 150)
    pages = int((-(-lengths // 16)).sum())
    cache, codes, scales = some_cache(gpu, pages, 16, 2, dim, fmt, 302)
    batch, plain, rows = some_batch(gpu, new.tolist(), lengths.tolist(), 16, pages, 303, columns, pad=3, first=2)
    got = form(kind, rows, 8, cache, batch)[0]
    assert got == CHUNK if columns else got in (TILES4, TILES8)
    q = dev(2 * W.normal((rows, 8, dim), 304, 1.0), gpu, TYPES[kind])
    few = slice(0, 8, 5)  # the oracle on heads 0 and 5, which read 0 and 1 of the cache
    want, size, total, reach = O.attention(host(q[:, few]), codes, scales, fmt, plain, window=40)
    tol = tight(kind, want, size, total, reach, dim, largest(scales, fmt))
    close("many", paged.attention(q, cache, batch, window=40)[:, few], want, tol)


def largest(scales, fmt):
    """What a value of each column can be."""
    return np.exp2(scales[1].max((0, 1, 2)) - 127.0).repeat(32) * (448 if fmt == "fp8" else 6)


def guarded(shape, dtype, gpu):
    """A tensor inside a larger one of known bytes, and a check that these are as they were."""
    size = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    around = torch.full((size + (2 << 20),), 0x5a, dtype=torch.uint8, device=gpu)
    inside = around[1 << 20:(1 << 20) + size].view(dtype).view(shape)

    def intact():
        return bool((around[:1 << 20] == 0x5a).all() and (around[(1 << 20) + size:] == 0x5a).all())

    return inside, intact


def call(name, *args):
    assert _native.check(getattr(_native.lib(), name)(*args, torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,columns", [(4, 5), (40, 9000)])
def test_starts_and_lengths_without_order(gpu, heads, columns, kind):
    """Starts below 0, behind the rows and before the one before, lengths below 0 and of 2^31 - 1: rows that only one
    sequence claims have their results, and nothing outside the tensors is touched."""
    dtype, rows, kv, dim = TYPES[kind], 40, 2, 64
    cache, codes, scales = some_cache(gpu, 20, 16, kv, dim, "fp8", 311)
    table = np.full((4, columns), -1, np.int32)
    table[:, :5] = np.random.default_rng(312).permutation(20).reshape(4, 5)
    wild = paged.Batch(ints([-7, 5, 12, 9, 2 ** 31 - 1], gpu), ints([20, -4, 30, 2 ** 31 - 1], gpu),
                       torch.from_numpy(table.copy()).to(gpu))
    # Rows 0..4 at 15..19 of the first, 5..8 below 0 of the second, 12..39 at 12..39 of the fourth; 9..11 of two.
    plain = (np.array([0, 5, 9, 12, 40]), np.array([20, 0, 0, 40]), table)
    sure = np.r_[0:9, 12:40]
    assert (form(kind, rows, heads, cache, wild)[0] == CHUNK) == (heads == 40)
    k, v = (dev(W.normal((rows, kv, dim), s, 1.0), gpu, dtype) for s in (313, 314))
    q = dev(W.normal((rows, heads, dim), 315, 1.0), gpu, dtype)

    plan = paged.rotary_plan(dim, device=gpu)
    out, intact = guarded((rows, heads, dim), dtype, gpu)
    call("ancha_paged_rotary", q.data_ptr(), list(TYPES).index(kind), rows, heads, dim, heads * dim, dim, None, 0,
         wild._at, plan._at, out.data_ptr())
    at = np.zeros(rows)
    for r, _, position in O.rows_of(plain, rows):
        at[r] = position
    at[5:9] = np.arange(5, 9) - 12
    want = O.rotate(host(q), at, plan.freqs.tolist())
    close("rotary", out[sure], want[sure], rotary_tolerance(host(q), plan, want, dtype)[sure])
    assert intact()

    both = [guarded(t.shape, torch.uint8, gpu) for t in (cache.codes, cache.scales)]
    for (t, _), a in zip(both, (codes, scales)):
        t.copy_(torch.from_numpy(a))
    cache = paged.Cache(both[0][0], both[1][0], "fp8")
    assert cache.write(k, v, wild) is cache
    O.write(codes, scales, "fp8", host(k), host(v), plain)
    for (t, intact), a in zip(both, (codes, scales)):
        got = t.cpu().numpy()
        for position in (9, 10, 11):  # of the rows claimed twice
            to = O.place(plain, 3, position, 20, 16)
            a[:, to[0], :, to[1]] = got[:, to[0], :, to[1]]
        assert np.array_equal(got, a) and intact()

    need = _native.lib().ancha_paged_attention_workspace(list(TYPES).index(kind), rows, heads, cache._at, wild._at)
    for window in (0, 9):
        out, intact = guarded((rows, heads, dim), dtype, gpu)
        space, whole = guarded((max(need, 16),), torch.uint8, gpu)
        call("ancha_paged_attention", q.data_ptr(), list(TYPES).index(kind), rows, heads, heads * dim, dim, cache._at,
             wild._at, ctypes.c_double(0.125), 1, window, space.data_ptr(), need, out.data_ptr())
        want, size, total, reach = O.attention(host(q), codes, scales, "fp8", plain, window=window or None)
        tol = tight(kind, want, size, total, reach, dim, largest(scales, "fp8"))
        close(f"attention {window}", out[sure], want[sure], tol[sure])
        assert intact() and whole()

    size = 5 * 16 + 7
    (rk, one), (rv, two) = (guarded((4, size, kv, dim), dtype, gpu) for _ in (0, 1))
    call("ancha_paged_read", cache._at, wild._at, size, list(TYPES).index(kind), rk.data_ptr(), rv.data_ptr())
    held = (plain[0], np.array([20, 0, 30, size]), table)
    for i in range(4):
        want = O.sequence(codes, scales, "fp8", held, i, size)
        for got, x in ((rk[i], want[0]), (rv[i], want[1])):
            assert torch.equal(got.cpu(), torch.from_numpy(x).to(dtype))
    assert one() and two()


@pytest.mark.parametrize("heads,columns", [(4, 5), (40, 9000)])
def test_more_tiles_than_rows_can_have(gpu, heads, columns):
    """A hundred sequences that all claim all rows: the tiles that are computed are those of the call, no more."""
    rows = 40
    cache, codes, scales = some_cache(gpu, 5, 16, 2, 64, "fp8", 321)
    table = np.full((100, columns), -1, np.int32)
    table[:, :5] = np.arange(5)
    wild = paged.Batch(ints([0, rows] * 50 + [0], gpu), ints([70] * 100, gpu), torch.from_numpy(table).to(gpu))
    q = dev(W.normal((rows, heads, 64), 322, 1.0), gpu, torch.bfloat16)
    need = _native.lib().ancha_paged_attention_workspace(2, rows, heads, cache._at, wild._at)
    out, intact = guarded((rows, heads, 64), torch.bfloat16, gpu)
    space, whole = guarded((max(need, 16),), torch.uint8, gpu)
    call("ancha_paged_attention", q.data_ptr(), 2, rows, heads, heads * 64, 64, cache._at, wild._at,
         ctypes.c_double(0.125), 1, 0, space.data_ptr(), need, out.data_ptr())
    torch.cuda.synchronize()
    assert intact() and whole()
