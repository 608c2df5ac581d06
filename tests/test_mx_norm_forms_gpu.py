"""The row norm into codes in every form that the rule on rows and columns picks, against the 64-bit oracle: the
kernel evaluates in 64 bits, so the bytes have to be equal. From 1024 rows on narrow rows share a wave or a
workgroup; 1030 rows leave the last one partly empty."""
import numpy as np
import pytest
import torch

from ancha_amd import _native, mx
from ancha_amd import workload as W
from oracle import mx as O
from tests.test_mx_gpu import TYPES, dev, host, rows_of, same_bytes

pytestmark = pytest.mark.gpu

# rows, columns: 16, 32, 64 and 128 threads a row; then the forms of few rows and of long ones.
SHAPES = [(1030, 1), (1030, 100), (1025, 200), (1030, 384), (1037, 500), (1030, 700), (1030, 768), (1029, 1000),
          (1024, 1024), (1030, 1549), (1030, 2048), (1030, 2500), (7, 384), (1023, 128), (37, 1549), (5, 2500),
          (5, 5000), (5, 12000), (4, 17000)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_norms(gpu, rows, dim, kind):
    """Both norms with rows of zeros, infinities, NaN and sums that overflow fp16 among ordinary ones."""
    dtype = TYPES[kind]
    x, r = dev(rows_of((rows, dim), 7) * 0.01, gpu, dtype), dev(W.normal((rows, dim), 8, 1.0), gpu, dtype)
    g = dev(np.sqrt(dim) * (1 + 0.3 * W.normal((dim,), 9, 1.0)), gpu)
    x[0] = 0
    x[1, dim // 2], x[2, dim - 1], x[rows - 1, 0] = float("inf"), float("nan"), float("-inf")
    x[3, dim - 1] = r[3, dim - 1] = 60000
    for fmt, eps, scale in (("fp8", 1e-5, None), ("fp4", 0.0, g)):
        s = None if scale is None else host(scale)
        same_bytes(f"norm {rows} x {dim} {fmt}", mx.unit_norm(x, scale, eps, fmt),
                   O.encode(O.unit_norm(host(x), s, eps), fmt))
        got, total = mx.add_unit_norm(x, r, scale, eps, fmt)
        h = (x.float() + r.float()).to(dtype)
        assert torch.equal(total.nan_to_num(nan=-7.0), h.nan_to_num(nan=-7.0))
        same_bytes(f"add norm {rows} x {dim} {fmt}", got, O.encode(O.unit_norm(host(h), s, eps), fmt))


@pytest.mark.parametrize("rows,dim", [s for s in SHAPES if s[1] > 1])
def test_strides_and_sums_in_place(gpu, rows, dim):
    """Rows apart and off their alignment; the sum in place of either operand; nothing behind the last row."""
    lib, stream = _native.lib(), torch.cuda.current_stream().cuda_stream
    base, other = dev(rows_of((rows, dim + 5), 13), gpu), dev(W.normal((rows, dim + 9), 14, 2.0), gpu)
    x, r = base[:, 3:dim + 3], other[:, 2:dim + 2]
    want = x + r
    codes = O.encode(O.unit_norm(host(want)), "fp8")
    got, total = mx.add_unit_norm(x, r)
    assert torch.equal(total, want) and total.is_contiguous()
    same_bytes("strided", got, codes)
    pitch, blocks = lib.ancha_mx_pitch(dim, 8), lib.ancha_mx_scales(dim)
    for place in (0, 1):
        both = [torch.full((rows + 3, dim), 7.0, device=gpu) for _ in range(2)]
        both[0][:rows], both[1][:rows] = x, r
        c = torch.full((rows + 3, pitch), 7, dtype=torch.uint8, device=gpu)
        s = torch.full((rows + 3, blocks), 7, dtype=torch.uint8, device=gpu)
        rc = lib.ancha_mx_norm(both[0].data_ptr(), 0, rows, dim, dim, both[1].data_ptr(), dim, None, 0.0, 8,
                               both[place].data_ptr(), c.data_ptr(), s.data_ptr(), stream)
        assert rc == _native.OK and torch.equal(both[place][:rows], want)
        assert (both[place][rows:] == 7).all() and (c[rows:] == 7).all() and (s[rows:] == 7).all()
        assert np.array_equal(c[:rows].cpu().numpy(), codes[0])
        assert np.array_equal(s[:rows].cpu().numpy(), codes[1])
