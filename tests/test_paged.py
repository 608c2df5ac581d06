"""The paged operators without a GPU: frequencies, the oracle against a dense computation, every refusal that is made
before a launch, and what the built kernels keep in registers."""
import ctypes
import math
import os
import re
import subprocess
import sys
import tempfile
import textwrap

import numpy as np
import pytest
import torch

from ancha_amd import _native, paged
from oracle import mx as OM
from oracle import paged as O
from tests.test_wide_stores import OBJDUMP, code_objects


@pytest.fixture(scope="module")
def lib():
    l = _native.lib()
    if l.ancha_hip_available():
        pytest.skip("host-buffer argument checks run only where no gfx950 device is visible")
    return l


def test_frequencies():
    f, m = paged.frequencies(8, 10000.0)
    assert np.allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-15) and m == 1
    assert np.allclose(paged.frequencies(8, 10000.0, "linear", 4.0)[0], np.array(f) / 4, rtol=1e-15)
    g, m = paged.frequencies(8, 10000.0, "ntk", 4.0)
    assert g[0] == 1 and abs(g[3] - f[3] / 4) < 1e-15 * g[3] * 100 and m == 1
    g, m = paged.frequencies(8, 10000.0, "yarn", 4.0, 4096)
    turns = 4096 * np.array(f) / (2 * math.pi)  # 651.9, 65.2, 6.52, 0.65
    assert g[:2] == f[:2] and abs(g[3] - f[3] / 4) < 1e-18
    share = (turns[2] - 1) / 31
    assert abs(g[2] - f[2] * (share + (1 - share) / 4)) < 1e-17 and abs(m - (0.1 * math.log(4) + 1)) < 1e-15
    assert paged.frequencies(2, 500.0) == ([1.0], 1.0)
    for how, text in (((0,), "width"), ((3,), "width"), ((8, -1.0), "base"), ((8, float("inf")), "base"),
                      ((64, 2.0 ** -21), "2\\*\\*20"),
                      ((8, 1e4, "dynamic"), "scaling"), ((8, 1e4, "linear", 0.5), "factor"),
                      ((8, 1e4, None, 2.0), "factor"),
                      ((8, 1e4, "yarn", float("nan"), 5), "factor"), ((8, 1e4, "yarn", 2.0), "original"),
                      ((2, 1e4, "ntk", 2.0), "ntk")):
        with pytest.raises(ValueError, match=text):
            paged.frequencies(*how)


def test_oracle_against_a_dense_computation():
    rng = np.random.default_rng(1)
    dim, kv, page, pages, length, n = 64, 2, 16, 5, 37, 9
    k, v = rng.standard_normal((2, length, kv, dim))
    codes, scales = np.zeros((2, pages, kv, page, dim), np.uint8), np.zeros((2, pages, kv, page, 2), np.uint8)
    table = np.array([[4, 1, 2]])
    O.write(codes, scales, "fp8", k, v, (np.array([0, length]), np.array([length]), table))
    batch = (np.array([0, n]), np.array([length]), table)
    held = O.sequence(codes, scales, "fp8", batch, 0, length)
    for x, got in ((k, held[0]), (v, held[1])):
        want = OM.decode(*OM.encode(x.reshape(-1, dim), "fp8"), "fp8", dim).reshape(x.shape)
        assert np.array_equal(got, want)
    q = rng.standard_normal((n, 4, dim))
    out = O.attention(q, codes, scales, "fp8", batch, window=30)[0]
    kk, vv = (torch.from_numpy(h).repeat_interleave(2, 1).transpose(0, 1) for h in held[:2])
    s = torch.from_numpy(q).transpose(0, 1) @ kk.transpose(1, 2) / 8
    at, key = torch.arange(length - n, length)[:, None], torch.arange(length)
    s = s.masked_fill((key > at) | (key <= at - 30), -math.inf)
    want = (torch.softmax(s, 2) @ vv).transpose(0, 1).numpy()
    assert np.abs(out - want).max() < 1e-13
    x = rng.standard_normal((3, 2, 10))
    f = [1.0, 0.3, 0.01]
    for layout in ("half", "interleaved"):
        y = O.rotate(x, [0, 5, -7], f, layout, 1.5)
        first, second = ([0, 1, 2], [3, 4, 5]) if layout == "half" else ([0, 2, 4], [1, 3, 5])
        for r, p in enumerate((0, 5, -7)):
            for i, w in enumerate(f):
                a, b = x[r, :, first[i]], x[r, :, second[i]]
                assert np.allclose(y[r, :, first[i]], 1.5 * (a * math.cos(p * w) - b * math.sin(p * w)))
                assert np.allclose(y[r, :, second[i]], 1.5 * (b * math.cos(p * w) + a * math.sin(p * w)))
        assert np.array_equal(y[..., 6:], x[..., 6:])


def structures(p, **changes):
    b = dict(starts=p, lengths=p, table=p, sequences=2, columns=3)
    c = dict(codes=p, scales=p, pages=4, heads=2, page=16, dim=64, format=8)
    f = dict(freqs=p, width=64, interleaved=0, magnitude=1.0)
    for name, value in changes.items():
        kind, field = name.split("_", 1)
        {"b": b, "c": c, "f": f}[kind][field] = value
    return _native.PagedBatch(**b), _native.PagedCache(**c), _native.PagedPlan(**f)


def test_entry_points_check_arguments(lib):
    buf = ctypes.create_string_buffer(1 << 14)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    INV, UNS, OK = _native.INVALID, _native.UNSUPPORTED, _native.OK
    ref = ctypes.byref

    def rotary(x=p, t=0, rows=3, heads=2, dim=64, ld=128, ldh=64, at=p, size=4, out=p, batch=True, plan=True,
               **changes):
        b, _, f = structures(p, **changes)
        return lib.ancha_paged_rotary(x, t, rows, heads, dim, ld, ldh, at, size, ref(b) if batch else None,
                                      ref(f) if plan else None, out, None)

    def write(k=p, v=p, t=0, rows=3, ld=128, ldh=64, batch=True, cache=True, **changes):
        b, c, f = structures(p, **changes)
        return lib.ancha_paged_write(k, v, t, rows, ld, ldh, ld, ldh, ref(b) if batch else None, ref(f),
                                     ref(c) if cache else None, None)

    def read(size=5, t=0, k=p, v=p, batch=True, cache=True, **changes):
        b, c, _ = structures(p, **changes)
        return lib.ancha_paged_read(ref(c) if cache else None, ref(b) if batch else None, size, t, k, v, None)

    def attention(q=p, t=0, rows=3, heads=4, ld=256, ldh=64, scale=0.125, window=0, ws=p, size=1 << 40, out=p,
                  batch=True, cache=True, **changes):
        b, c, _ = structures(p, **changes)
        return lib.ancha_paged_attention(q, t, rows, heads, ld, ldh, ref(c) if cache else None,
                                         ref(b) if batch else None, scale, 1, window, ws, size, out, None)

    def refused(rc, code, text):
        assert rc == code and text in _native.last_error(), (rc, _native.last_error())

    # All in order: only the device is missing.
    for call in (rotary, write, read, attention):
        refused(call(), UNS, "gfx950")
        refused(call(t=3), INV, "type")
        refused(call(batch=False) if call is not rotary else call(batch=False, at=None), INV, "null batch")
        if call is not rotary:
            refused(call(cache=False), INV, "null cache")
            for change in ({"c_pages": 0}, {"c_heads": 0}, {"c_codes": None}, {"c_scales": None}):
                refused(call(**change), INV, "empty cache")
            refused(call(c_codes=p + 8), INV, "aligned")
            refused(call(c_scales=p + 4), INV, "aligned")
            refused(call(c_format=5), INV, "format")
            for page in (0, 8, 17, 48, 1 << 17):
                refused(call(c_page=page), UNS, "power of two")
            for dim in (0, 32, 96, 512):
                refused(call(c_dim=dim), UNS, "head width")
            refused(call(c_pages=1 << 31), UNS, "too large")
            refused(call(c_pages=1 << 30, c_page=65536, c_heads=4), UNS, "too large")
            refused(call(b_lengths=None), INV, "null tensor in the batch")
            refused(call(b_table=None), INV, "null tensor in the batch")
            refused(call(b_table=p + 2), INV, "aligned")
            refused(call(b_columns=1 << 31), UNS, "too many sequences")
            refused(call(b_sequences=(1 << 31) - 1), UNS, "too many sequences")
    for call in (rotary, write):
        for change in ({"f_freqs": None}, {"f_freqs": p + 4}):
            refused(call(**change), INV, "freqs")
        for width in (0, 3, 66):
            refused(call(f_width=width), INV, "width")
        for m in (0.0, -1.0, float("nan"), float("inf"), 1e39):
            refused(call(f_magnitude=m), INV, "magnitude")
        refused(call(ld=1 << 62), UNS, "too many")
        refused(call(rows=1 << 24), UNS, "too many")
        assert call(rows=0) == OK
    refused(rotary(plan=False), INV, "null plan")
    refused(rotary(at=p + 2), INV, "positions")
    refused(rotary(at=p + 4, size=8), INV, "positions")
    refused(rotary(size=2), INV, "positions")
    refused(rotary(at=None, b_starts=None), INV, "null tensor in the batch")
    refused(rotary(at=None, b_starts=p + 1), INV, "aligned")
    refused(rotary(at=None, b_table=None), UNS, "gfx950")  # not read
    refused(rotary(x=None), INV, "null tensor")
    refused(rotary(out=None), INV, "null tensor")
    refused(rotary(dim=4096, f_width=4096), UNS, "too many")
    refused(rotary(dim=4096, heads=1024), UNS, "too many")
    assert rotary(heads=0) == OK
    refused(write(k=None), INV, "null tensor")
    refused(write(v=None), INV, "null tensor")
    refused(write(b_starts=None), INV, "null tensor in the batch")
    refused(read(k=None), INV, "null tensor")
    refused(read(v=p + 8), INV, "aligned")
    refused(read(b_starts=None), UNS, "gfx950")  # not read
    refused(read(size=1 << 24), UNS, "too many")
    refused(read(size=1 << 31), UNS, "too many")
    assert read(size=0) == OK and read(b_sequences=0) == OK
    for heads in (0, 3):
        refused(attention(heads=heads), INV, "multiple")
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-31, 1e31):
        refused(attention(scale=scale), INV, "scale")
    refused(attention(q=None), INV, "null tensor")
    refused(attention(out=None), INV, "null tensor")
    refused(attention(rows=1 << 30), UNS, "too many")
    refused(attention(rows=1 << 26, heads=16), UNS, "too many")
    assert attention(rows=0) == OK
    # Long sequences are shared out, which takes a workspace: as much as the call itself asks for, of every type,
    # whatever kernel the sizes lead to (a tile of rows is another one for other types).
    for dim, rows, sequences, columns in ((64, 3, 2, 4096), (128, 32, 8, 64), (128, 64, 2, 512), (64, 100, 1, 512),
                                          (256, 9, 3, 512), (128, 300, 2, 512)):
        how = dict(b_columns=columns, b_sequences=sequences, c_dim=dim)
        b, c, _ = structures(p, **how)
        for t in (0, 1, 2):
            need = lib.ancha_paged_attention_workspace(t, rows, 8, ref(c), ref(b))
            assert need > 0
            call = dict(how, t=t, rows=rows, heads=8, ld=8 * dim, ldh=dim)
            refused(attention(size=need - 1, **call), INV, "workspace")
            refused(attention(ws=None, **call), INV, "workspace")
            refused(attention(ws=p + 8, **call), INV, "workspace")
            refused(attention(size=need, **call), UNS, "gfx950")
    for t, rows, heads in ((0, 0, 4), (0, 3, 3), (0, 3, 0), (3, 3, 4)):
        assert lib.ancha_paged_attention_workspace(t, rows, heads, ref(c), ref(b)) == 0
    assert lib.ancha_paged_attention_workspace(0, 3, 4, None, ref(b)) == 0
    assert lib.ancha_hip_check() == 0


def test_wrappers_reject_host_tensors_and_names():
    x, at = torch.zeros((4, 2, 64)), torch.zeros(4, dtype=torch.int32)
    codes = torch.zeros((2, 4, 2, 16, 64), dtype=torch.uint8)
    for call in (lambda: paged.rotary(x, at, None), lambda: paged.attention(x, None, None),
                 lambda: paged.Batch(at, at, at), lambda: paged.Cache(codes, codes, "fp8"),
                 lambda: paged.Rotary(torch.ones(4, dtype=torch.float64))):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    for call, text in ((lambda: paged.Cache(codes, codes, "fp6"), "format"),
                       (lambda: paged.Cache.empty(4, 16, 2, 96, device="cpu"), "dim"),
                       (lambda: paged.Rotary(torch.ones(4), "pairs"), "layout")):
        with pytest.raises(ValueError, match=text):
            call()


def test_kernels_keep_their_registers():
    """No kernel of the paged operators spills. (Where a group of sixteen accumulation registers is spilled in parts,
    this compiler has been seen to leave one of them out when it brings the group back.)"""
    readelf = os.path.join(os.path.dirname(OBJDUMP), "llvm-readelf")
    if not os.path.exists(readelf):
        pytest.skip("llvm-readelf is not installed")
    found = 0
    for code in code_objects(_native.LIB_PATH):
        if b"paged" not in code:
            continue
        with tempfile.NamedTemporaryFile(suffix=".co") as f:
            f.write(code)
            f.flush()
            notes = subprocess.run([readelf, "--notes", f.name], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("- .agpr_count:")[1:]:
            name = re.search(r"\.name:\s+(\S+)", kernel)[1]
            found += 1
            for what in ("vgpr_spill_count", "sgpr_spill_count", "private_segment_fixed_size"):
                assert int(re.search(rf"\.{what}:\s+(\d+)", kernel)[1]) == 0, f"{name}: {what}"
    assert found > 40


_CHILD = textwrap.dedent("""
import sys
sys.path.insert(0, sys.argv[1])
from ancha_amd import _native
lib, N = _native.lib(), None
calls = {
    "ancha_paged_rotary": lambda: lib.ancha_paged_rotary(N, 0, 4, 2, 64, 128, 64, N, 4, N, N, N, N),
    "ancha_paged_write": lambda: lib.ancha_paged_write(N, N, 0, 4, 128, 64, 128, 64, N, N, N, N),
    "ancha_paged_read": lambda: lib.ancha_paged_read(N, N, 4, 0, N, N, N),
    "ancha_paged_attention": lambda: lib.ancha_paged_attention(N, 0, 4, 2, 128, 64, N, N, 0.1, 1, 0, N, 0, N, N),
}
sizes = {"ancha_paged_attention_workspace"}
assert {n for n in _native.SIGNATURES if n.startswith("ancha_paged_")} == set(calls) | sizes
for name, call in calls.items():
    assert call() == -2, name
    assert "sticky device failure" in _native.last_error(), name
print("sticky", len(calls))
""")


def test_a_device_failure_is_sticky():
    """A HIP failure recorded once (injected at library load) is what every later call returns."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _CHILD, root], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ANCHA_HIP_INJECT_FAILURE="2"))
    assert r.returncode == 0 and "sticky 4" in r.stdout, r.stdout + r.stderr
