"""The microscaled operators without a GPU: the oracle's rounding against torch's own 8-bit type and
written-out values, row sizes, and every refusal that is made before a launch."""
import ctypes
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest
import torch

from ancha_amd import _native, fused, mx
from oracle import mx as O


@pytest.fixture(scope="module")
def lib():
    l = _native.lib()
    if l.ancha_hip_available():
        pytest.skip("host-buffer argument checks run only where no gfx950 device is visible")
    return l


def test_oracle_rounds_like_torch():
    v = np.concatenate((np.linspace(-460, 460, 9001), np.linspace(-0.05, 0.05, 4001),
                        (O.grid("fp8")[1:] + O.grid("fp8")[:-1]) / 2))
    v = np.clip(v, -448, 448).astype(np.float32)
    got = O.grid("fp8")[O.nearest(v.astype(np.float64), "fp8")]
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).float().abs().numpy()
    assert np.array_equal(got, want)


def test_oracle_known_blocks():
    x = np.zeros((1, 40), np.float32)
    x[0, :9] = [6, -5, 2.5, 0.25, 0.75, 7.9, 1.75, -0.2, 3.5]
    codes, scales = O.encode(x, "fp4")
    assert scales[0].tolist() == [127, 0, 0, 0]
    low = [c for b in codes[0, :5] for c in (b & 15, b >> 4)][:9]
    #         6   -5->-4   2.5->2  .25->0  .75->1  7.9->6  1.75->2  -.2->-0  3.5->4
    assert low == [7, 8 + 6, 4, 0, 2, 7, 4, 8, 6]
    x = np.array([[1.0, np.inf] + [0.0] * 30 + [2.0 ** -140] * 3], np.float32)
    codes, scales = O.encode(x, "fp8")
    assert scales[0].tolist() == [255, 0, 0, 0]
    values = O.decode(codes, scales, "fp8", 35)
    assert np.isnan(values[0, :32]).all() and (values[0, 32:] == 0).all()


@pytest.mark.parametrize("dim,groups", [(0, 0), (1, 1), (128, 1), (129, 2), (8192, 64)])
def test_row_sizes(dim, groups):
    l = _native.lib()
    assert l.ancha_mx_pitch(dim, 8) == 128 * groups
    assert l.ancha_mx_pitch(dim, 4) == 64 * groups
    assert l.ancha_mx_scales(dim) == 4 * groups
    assert l.ancha_mx_pitch(dim, 7) == 0


@pytest.mark.parametrize("k,m,size", [(1, 1, 2 * 4352), (128, 128, 2 * 4352), (129, 129, 8 * 4352),
                                      (384, 1664, 26 * 3 * 4352), (0, 5, 0), (5, 0, 0),
                                      (1 << 20, 1 << 20, 0), (128, (1 << 24) + 1, 0),
                                      ((1 << 23) + 1, 64, 0), (128, 1 << 24, (1 << 18) * 4352)])
def test_weight_sizes(k, m, size):
    assert _native.lib().ancha_mx_weight_bytes(k, m) == size


def test_entry_points_check_arguments(lib):
    buf = ctypes.create_string_buffer(1 << 14)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    INV, UNS = _native.INVALID, _native.UNSUPPORTED
    q = lambda x=p, t=0, r=2, d=40, ld=40, f=8, c=p, s=p: lib.ancha_mx_quantize(  # noqa: E731
        x, t, r, d, ld, f, c, s, None)
    for rc, text in ((q(t=3), "type"), (q(f=5), "format"), (q(ld=39), "stride"), (q(x=None), "null"),
                     (q(c=None), "null"), (q(s=None), "null"), (q(c=p + 8), "aligned"), (q(s=p + 2), "aligned")):
        assert rc == INV
    q(c=p + 8)
    assert "aligned" in _native.last_error()
    assert q(r=0) == _native.OK and q(d=0, ld=0) == _native.OK
    assert q(r=1 << 30, d=1 << 20, ld=1 << 20) == UNS and "too many" in _native.last_error()
    assert q() == UNS and "gfx950" in _native.last_error()  # all in order: only the device is missing
    n = lambda r=p, ldr=40, total=p, eps=0.0, x=p, ldx=40: lib.ancha_mx_norm(  # noqa: E731
        x, 0, 2, 40, ldx, r, ldr, None, eps, 8, total, p, p, None)
    assert n(ldr=39) == INV and n(total=None) == INV and n(eps=-1.0) == INV
    assert n(eps=float("nan")) == INV and n(eps=float("inf")) == INV
    assert n(r=p + 64, total=p, ldx=44) == INV and "contiguous" in _native.last_error()
    assert n(r=None, total=None) == UNS and n() == UNS
    v = lambda c=p, o=p, f=4, t=2: lib.ancha_mx_values(c, p, 2, 40, f, t, o, None)  # noqa: E731
    assert v(c=None) == INV and v(o=None) == INV and v(f=1) == INV and v(t=-1) == INV and v() == UNS
    w = lambda x=p, k=40, m=8, o=p: lib.ancha_mx_weight(x, 0, k, m, 8, 1, o, None)  # noqa: E731
    assert w(x=None) == INV and w(o=p + 4) == INV and w(k=0) == UNS and w(m=0) == UNS and w() == UNS
    y = lambda c=p, n=4, k=40, f=8, wt=p, m=128, rope=None, tok=0, width=0, t=0, of=0, o=p, os=None: \
        lib.ancha_mx_linear(c, p, n, k, f, wt, m, None, 0, rope, tok, width, None, t, of, o, os,
                                None)  # noqa: E731
    assert y(c=None) == INV and y(wt=None) == INV and y(o=None) == INV and y(f=3) == INV and y(t=9) == INV
    assert y(of=8) == INV and y(of=5) == INV and y(of=8, t=1, os=p) == INV and y(wt=p + 4) == INV
    assert y(k=0) == UNS and y(m=0) == UNS and y(n=0) == _native.OK
    for tok, width in ((0, 64), (3, 64), (4, 32), (4, 128)):
        assert y(rope=p, tok=tok, width=width) == UNS and "rotary" in _native.last_error()
    assert y(m=(1 << 24) + 1) == UNS and y(k=(1 << 23) + 1) == UNS
    assert y(n=(1 << 31) - 1) == UNS and "too many" in _native.last_error()
    assert y() == UNS and "gfx950" in _native.last_error()
    assert lib.ancha_hip_check() == 0


def test_wrappers_reject_host_tensors_and_names():
    x = torch.zeros((4, 64))
    for call in (lambda: mx.quantize(x), lambda: mx.unit_norm(x), lambda: mx.add_unit_norm(x, x),
                 lambda: mx.weight(x)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    with pytest.raises(ValueError, match="format"):
        mx.quantize(x, "fp6")
    with pytest.raises(ValueError, match="on a GPU"):
        mx.Tensor(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 4), dtype=torch.uint8), "fp4",
                  (4, 64))
    with pytest.raises(ValueError, match="microscaled"):
        mx.linear(x, x)
    with pytest.raises(ValueError, match="residual"):
        mx.add_unit_norm(x, None)
    assert fused.Epilogue().empty()


_CHILD = textwrap.dedent("""
import sys
sys.path.insert(0, sys.argv[1])
from ancha_amd import _native
lib, N = _native.lib(), None
calls = {
    "ancha_mx_quantize": lambda: lib.ancha_mx_quantize(N, 0, 4, 64, 64, 8, N, N, N),
    "ancha_mx_norm": lambda: lib.ancha_mx_norm(N, 0, 4, 64, 64, N, 0, N, 0.0, 8, N, N, N, N),
    "ancha_mx_values": lambda: lib.ancha_mx_values(N, N, 4, 64, 8, 0, N, N),
    "ancha_mx_weight": lambda: lib.ancha_mx_weight(N, 0, 64, 64, 1, 64, N, N),
    "ancha_mx_weight_values": lambda: lib.ancha_mx_weight_values(N, 64, 64, 0, N, N),
    "ancha_mx_linear": lambda: lib.ancha_mx_linear(N, N, 4, 64, 8, N, 64, N, 0, N, 0, 0, N, 0, 0, N, N, N),
}
sizes = {"ancha_mx_pitch", "ancha_mx_scales", "ancha_mx_weight_bytes"}
assert {n for n in _native.SIGNATURES if n.startswith("ancha_mx_")} == set(calls) | sizes
for name, call in calls.items():
    assert call() == -2, name
    assert "sticky device failure" in _native.last_error(), name
assert lib.ancha_mx_scales(64) == 4
print("sticky", len(calls))
""")


def test_a_device_failure_is_sticky():
    """A HIP failure recorded once (injected at library load) is what every later call returns."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _CHILD, root], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ANCHA_HIP_INJECT_FAILURE="2"))
    assert r.returncode == 0 and "sticky 6" in r.stdout, r.stdout + r.stderr
