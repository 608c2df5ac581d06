"""The product of microscaled rows where its forms and its roundings meet hard values: sums whose large
products cancel, GELU of infinities and far below zero. Oracle and tolerances: tests/test_mx_gpu.py."""
import math

import numpy as np
import pytest
import torch

from ancha_amd import fused, mx
from ancha_amd import workload as W
from oracle import mx as O
from tests.test_mx_gpu import (TYPES, check_codes, dev, expected, host, near, product_bound, rows_of,
                               same_bytes)

pytestmark = pytest.mark.gpu

# One size for each form of the product: few rows (16 and 32 a workgroup), 64 x 64 tiles with the steps in one
# chain and in four, 128 x 128 tiles, 256 columns.
FORMS = [(5, 300, 40), (24, 2100, 4200), (801, 1000, 1549), (130, 2100, 2050), (2100, 200, 1549), (8200, 130, 2048)]


def cancelling(n, k, m):
    """x [n, k], w [k, m] that both formats hold exactly: of every eight neighbouring products two are large and
    add up to 0, one is small, the others are 0."""
    rng = np.random.default_rng(n + k + m)
    x, w = np.zeros((n, k), np.float32), np.zeros((k, m), np.float32)
    large, small = O.grid("fp8")[-7:], O.grid("fp8")[1:41]  # 256 .. 448, 2^-9 .. 0.25
    for k0 in range(0, k - 7, 8):
        a, b, c = k0 + rng.choice(8, 3, replace=False)
        x[:, a] = rng.choice(large, n)
        x[:, b] = -x[:, a]
        x[:, c] = rng.choice(small, n)
        w[a] = w[b] = rng.choice((4.0, -4.0, 6.0, -6.0), m)
        w[c] = rng.choice((0.5, 1.0, 1.5), m)
    return x, w


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,m", FORMS)
def test_large_products_cancel(gpu, n, k, m, kind):
    """e4m3 sums are held in 32 bits whatever the result's type: small products beside large ones that cancel
    are what is left."""
    x, w = cancelling(n, k, m)
    t, handle = mx.quantize(dev(x, gpu), "fp8"), mx.weight(dev(w, gpu))
    xv, wv = host(t.values()), host(handle.values())
    y, tol = expected(xv, wv, "fp8", False, dtype=TYPES[kind])
    assert (tol < 0.25 * np.abs(y).mean()).all()
    near(f"{n}x{k}x{m} {kind}", host(mx.linear(t, handle, dtype=TYPES[kind])), y, tol)


# ---- GELU. Rows of zeros give products of exactly 0, so the bias is what GELU takes.

GELU_FORMS = [(3, 200, 700), (24, 2100, 4200), (801, 200, 1549), (130, 2100, 2050), (2100, 200, 1549), (8200, 130, 2048)]


def on_bias(gpu, n, k, m, values):
    zeros = mx.quantize(torch.zeros((n, k), device=gpu), "fp8")
    bias = torch.zeros(m, device=gpu)
    bias[:len(values)] = dev(values, gpu)
    return zeros, mx.weight(dev(np.ones((k, m)), gpu)), fused.Epilogue(bias=bias, gelu=True), host(bias)


@pytest.mark.parametrize("n,k,m", GELU_FORMS)
def test_gelu_of_infinities_in_codes(gpu, n, k, m):
    """GELU(-inf) = 0 leaves its block as it is, +inf and NaN spoil theirs."""
    values = np.ones(160, np.float32)
    values[5], values[32:64], values[70], values[100] = -np.inf, -np.inf, np.inf, np.nan
    t, w, e, bias = on_bias(gpu, n, k, m, values)
    y = np.where(bias == -np.inf, 0.0, O.gelu(np.where(np.isfinite(bias), bias, 0.0)))
    y = np.where(np.isnan(bias) | (bias == np.inf), bias, y)
    for fmt in ("fp8", "fp4"):
        want = O.encode(np.repeat(y[None], n, 0), fmt)
        assert want[1][0, :5].tolist().count(255) == 2 and want[1][0, 1] == 0
        same_bytes(fmt, mx.linear(t, w, e, format=fmt), want)
    for dtype in TYPES.values():
        got = mx.linear(t, w, e, dtype=dtype).float()
        assert (got[:, 32:64] == 0).all() and (got[:, 5] == 0).all() and (got[:, 70] == float("inf")).all()
        assert got[:, 100].isnan().all() and int(got.isnan().sum()) == n


def gelu_error(x, dtype):
    """The kernel's documented error of GELU relative to its value."""
    steps = (1e-6, 4e-6, 1e-4, 2e-3) if dtype == torch.float32 else (2.5e-6, 3e-5, 1e-3, 3e-3)
    ends = (-2, -4, -6) if dtype == torch.float32 else (-2, -4, -8)
    return np.select([x >= e for e in ends], steps[:3], steps[3])


@pytest.mark.parametrize("n,k,m", GELU_FORMS)
def test_gelu_far_below_zero(gpu, n, k, m):
    """Results of 1e-34 to 3, neighbouring columns alike, so that blocks hold nothing but small ones."""
    t, w, e, bias = on_bias(gpu, n, k, m, np.linspace(-12.5, 3, min(m, 1500)).astype(np.float32))
    y = 0.5 * bias * np.array([math.erfc(-b / math.sqrt(2)) for b in bias])
    y = np.repeat(y[None], n, 0)
    for kind, dtype in TYPES.items():
        type_off = torch.finfo(dtype).eps / 2 * np.abs(y) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        near(f"{n}x{k}x{m} {kind}", host(mx.linear(t, w, e, dtype=dtype)), y,
             gelu_error(bias, dtype) * np.abs(y) * (1 + torch.finfo(dtype).eps) + type_off)
    for fmt in ("fp8", "fp4"):
        got = mx.linear(t, w, e, format=fmt)
        check_codes(f"{n}x{k}x{m} {fmt}", got, y, gelu_error(bias, torch.bfloat16) * np.abs(y), fmt)


# ---- Every form with every epilogue; rows of whole groups of four columns and others.

EPILOGUE_SIZES = [(5, 300, 40), (13, 300, 327), (24, 2100, 4200), (29, 2100, 4101), (801, 1000, 1549), (800, 200, 1552),
                  (130, 2100, 2050), (130, 2100, 2052), (2100, 200, 1549), (2100, 130, 1600), (8200, 130, 2047),
                  (8200, 160, 2048), (3, 130, 20000), (16, 300, 33001), (40, 130, 30000)]


def result(x, w, bias, gelu, residual, dtype=None):
    """The 64-bit result and how far the kernel's, in `dtype` or before it becomes codes, may be from it (GELU's
    slope is at most 1.13)."""
    off = product_bound(x, w, "fp8", False) + 1e-37
    y = x @ w + bias
    off += 2.0 ** -24 * (np.abs(y) + off)
    if gelu:
        value = (0.5 * torch.special.erfc(torch.from_numpy(-y / math.sqrt(2)))).numpy() * y
        off = 1.13 * off + gelu_error(y - off, dtype) * (np.abs(value) + 1.13 * off)
        y = value
    if residual is not None:
        y = y + residual
        off = off + 2.0 ** -24 * (np.abs(y) + off)
    if dtype is None:
        return y, off
    half = torch.finfo(dtype).eps / 2
    return y, off + half * (np.abs(y) + off) + float(torch.finfo(dtype).smallest_normal) * half


def rows_times_weight(gpu, n, k, m, seed):
    """Rows of e4m3 codes with large channels and blocks of very different size, a weight, and their values."""
    t = mx.quantize(dev(rows_of((n, k), seed), gpu), "fp8")
    w = mx.weight(dev(W.normal((k, m), seed + 1, 1 / np.sqrt(k)), gpu))
    return t, w, host(t.values()), host(w.values())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,m", EPILOGUE_SIZES)
def test_values(gpu, n, k, m, kind):
    dtype = TYPES[kind]
    t, w, x, wv = rows_times_weight(gpu, n, k, m, 31)
    b, r = dev(W.normal((m,), 33, 1.0), gpu), dev(W.normal((n, m), 34, 2.0), gpu, dtype)
    for gelu, residual in ((False, None), (True, r)):
        got = mx.linear(t, w, fused.Epilogue(bias=b, gelu=gelu, residual=residual), dtype=dtype)
        near(f"{n}x{k}x{m} {kind} gelu {gelu}", host(got),
             *result(x, wv, host(b), gelu, None if residual is None else host(r), dtype))


@pytest.mark.parametrize("out", ["fp8", "fp4"])
@pytest.mark.parametrize("n,k,m", EPILOGUE_SIZES)
def test_codes(gpu, n, k, m, out):
    t, w, x, wv = rows_times_weight(gpu, n, k, m, 41)
    b, r = dev(W.normal((m,), 43, 1.0), gpu), dev(W.normal((n, m), 44, 2.0), gpu)
    for gelu, residual in ((True, None), (False, r)):
        got = mx.linear(t, w, fused.Epilogue(bias=b, gelu=gelu, residual=residual), format=out)
        y, tol = result(x, wv, host(b), gelu, None if residual is None else host(r))
        check_codes(f"{n}x{k}x{m} {out} gelu {gelu}", got, y, tol, out)


@pytest.mark.parametrize("n,k,m", EPILOGUE_SIZES)
def test_blocks_that_are_not_finite(gpu, n, k, m):
    """A NaN block of a row spoils that row alone, one of the weight its column alone, in values and in codes."""
    x, w = W.normal((n, k), 51, 1.0), W.normal((k, m), 52, 0.1)
    x[1, k - 1], x[n - 1, 40], w[70, m // 2] = np.inf, np.nan, np.nan
    t, handle = mx.quantize(dev(x, gpu), "fp8"), mx.weight(dev(w, gpu))
    want = torch.zeros((n, m), dtype=torch.bool, device=gpu)
    want[1], want[n - 1], want[:, m // 2] = True, True, True
    e = fused.Epilogue(bias=dev(W.normal((m,), 53, 1.0), gpu), gelu=True)
    for dtype in TYPES.values():
        assert torch.equal(mx.linear(t, handle, e, dtype=dtype).isnan(), want)
    blocks = torch.nn.functional.pad(want, (0, O.padded(m) - m)).view(n, -1, 32).any(2)
    for fmt in ("fp8", "fp4"):
        got = mx.linear(t, handle, e, format=fmt)
        assert torch.equal(got.scales == 255, blocks)
        assert torch.equal(got.values().isnan(), blocks.repeat_interleave(32, 1)[:, :m])


@pytest.mark.parametrize("n,k,m", EPILOGUE_SIZES)
def test_rotary(gpu, n, k, m):
    """Rotated query and key columns (where the width has any) at positions that start anew in the middle of
    tiles."""
    width = m // 128 * 64
    if not width:
        assert mx.linear(*rows_times_weight(gpu, n, k, m, 61)[:2],
                         fused.Epilogue(rotary=(torch.zeros((4, 1, 64), device=gpu), 64))) is None
        return
    tokens = max(d for d in range(1, 900) if n % d == 0)
    table = W.axis_rope_packed(W.rope_freqs(), tokens)
    t, w, x, wv = rows_times_weight(gpu, n, k, m, 61)
    b = dev(W.normal((m,), 63, 1.0), gpu)
    e = fused.Epilogue(bias=b, rotary=(dev(table, gpu), width))
    for kind, dtype in TYPES.items():
        y, tol = expected(x, wv, "fp8", False, host(b), rotary=(table.astype(np.float64), width), dtype=dtype)
        near(f"{n}x{k}x{m} {kind}", host(mx.linear(t, w, e, dtype=dtype)), y, tol)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,m", FORMS)
def test_rows_of_4_bits(gpu, n, k, m, kind):
    t = mx.quantize(dev(rows_of((n, k), 71), gpu), "fp4")
    w = mx.weight(dev(W.normal((k, m), 72, 1 / np.sqrt(k)), gpu))
    y, tol = expected(host(t.values()), host(w.values()), "fp4", False, dtype=TYPES[kind])
    near(f"{n}x{k}x{m} {kind}", host(mx.linear(t, w, dtype=TYPES[kind])), y, tol)


@pytest.mark.parametrize("pair", [448.0, 1.875])
@pytest.mark.parametrize("n,m", [(127, 8), (889, 1544)])
def test_each_product_beside_the_largest(gpu, n, m, pair):
    """Beside two products that cancel (the largest there are, the largest of small rows' values), every product
    of an e4m3 and an e2m1 code that stands in the same eight is left as it is."""
    values, factors = O.grid("fp8"), O.grid("fp4")
    x, w = np.zeros((n, 40), np.float32), np.zeros((40, m), np.float32)
    x[:, 0], x[:, 5], x[:, 31] = pair, -pair, 448  # the last one holds the block's scale, times 0
    w[0], w[5], w[12] = 6, 6, 6
    x[:, 3], w[3] = np.resize(values, n), np.resize(factors, m)
    t, handle = mx.quantize(dev(x, gpu), "fp8"), mx.weight(dev(w, gpu))
    assert np.array_equal(host(t.values()), x) and np.array_equal(host(handle.values()), w)
    assert np.array_equal(host(mx.linear(t, handle)), np.outer(x[:, 3].astype(np.float64), w[3]))


def test_weights_check_what_they_are_made_of(gpu):
    w = mx.weight(dev(W.normal((130, 70), 91, 1.0), gpu))
    t = mx.quantize(dev(W.normal((3, 130), 92, 1.0), gpu))
    assert torch.equal(mx.linear(t, mx.Weight(w._data.clone(), 130, 70)), mx.linear(t, w))
    for data, k, m in ((w._data[:-16], 130, 70), (w._data, 300, 70), (w._data.view(2, -1), 130, 70),
                       (w._data.view(torch.int8), 130, 70)):
        with pytest.raises(ValueError, match="data must"):
            mx.Weight(data, k, m)
