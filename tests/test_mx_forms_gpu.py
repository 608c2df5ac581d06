"""The product of microscaled rows where its forms and its roundings meet hard values: sums whose large
products cancel, GELU of infinities and far below zero. Oracle and tolerances: tests/test_mx_gpu.py."""
import math

import numpy as np
import pytest
import torch

from ancha_amd import fused, mx
from oracle import mx as O
from tests.test_mx_gpu import TYPES, check_codes, dev, expected, host, near, same_bytes

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
