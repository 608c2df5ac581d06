"""Which kernel a microscaled product or norm takes, where that was chosen by measurement (CPU; the rule counts the CUs
of the current device, 256 where there is none), and that the GPU tests' sizes reach every one."""
import pytest
import torch

from ancha_amd import _native, mx
from tests import test_mx_forms_gpu as G
from tests import test_mx_norm_forms_gpu as N

FEW16, FEW32, TILES64, CHAINS64, TILES128, TILES256 = range(6)


def form(n, k, m):
    return _native.lib().ancha_amd_mx_linear_form(n, k, m)


RULE = [
    # One tile of rows: the weight is read once, whatever its width.
    (1, 128, 32, FEW16), (1, 4096, 4096, FEW16), (16, 4096, 7168, FEW16), (8, 8192, 8224, FEW16),
    (1, 4096, 14336, FEW16), (16, 4096, 28672, FEW16), (1, 4096, 128256, FEW16), (16, 128, 1 << 24, FEW16),
    # Few rows of few columns: sixteen rows a workgroup while these fit one to a CU, then 32 for a long k.
    (24, 4096, 4096, FEW16), (128, 2048, 512, FEW16), (4096, 384, 32, FEW16), (17, 4096, 4128, FEW32),
    (24, 4096, 7168, FEW32), (32, 8192, 8192, FEW32), (24, 8192, 8160, FEW32), (64, 4096, 4096, FEW32),
    (64, 2048, 4096, FEW32), (64, 2047, 4096, FEW16), (64, 1024, 4096, FEW16), (128, 384, 1536, FEW16),
    (48, 4096, 4128, FEW16), (33, 4096, 5120, FEW16),
    # 64 x 64 tiles, four chains of steps while the tiles fit one to a CU and k is long.
    (24, 8192, 8224, CHAINS64), (24, 4096, 14336, CHAINS64), (64, 4096, 7168, CHAINS64),
    (128, 4096, 4096, CHAINS64), (512, 2048, 2048, CHAINS64), (512, 1024, 1024, TILES64),
    (17, 4096, 28672, TILES64), (64, 4096, 128256, TILES64), (128, 4096, 14336, TILES64),
    (512, 4096, 4096, TILES64), (801, 1000, 1549, TILES64), (2048, 1024, 1024, TILES64),
    # Larger ones.
    (65, 4096, 28672, TILES128), (128, 4096, 28672, TILES128), (1024, 4096, 4096, TILES128),
    (2048, 4096, 4096, TILES128), (96120, 1536, 384, TILES128), (4096, 4096, 4096, TILES256),
    (8192, 8192, 8192, TILES256), (96120, 384, 1536, TILES256),
]


@pytest.mark.parametrize("n,k,m,want", RULE)
def test_form_of_a_product(n, k, m, want):
    assert form(n, k, m) == want


@pytest.mark.parametrize("sizes", ["FORMS", "GELU_FORMS", "EPILOGUE_SIZES"])
def test_sizes_of_the_gpu_tests_reach_every_form(sizes):
    assert {form(*s) for s in getattr(G, sizes)} == set(range(6))


# rows, columns, threads a row, pieces of eight values of each (0, 0: rows read twice)
NORMS = [(1, 1, 64, 1), (1023, 512, 64, 1), (1023, 513, 256, 1), (1, 2048, 256, 1), (1, 2049, 256, 2),
         (5000, 4096, 256, 2), (1, 4097, 256, 4), (1, 8193, 512, 4), (9999, 16384, 512, 4), (1, 16385, 0, 0),
         (1024, 128, 16, 1), (1024, 129, 16, 2), (96120, 384, 16, 3), (1024, 512, 16, 4), (1024, 513, 32, 3),
         (1024, 768, 32, 3), (1024, 769, 64, 2), (1024, 1024, 64, 2), (6007, 1549, 128, 2), (1024, 2048, 128, 2)]


@pytest.mark.parametrize("rows,dim,threads,pieces", NORMS)
def test_form_of_a_norm(rows, dim, threads, pieces):
    assert _native.lib().ancha_amd_mx_norm_form(rows, dim) == 8 * threads + pieces
    assert 8 * threads * pieces >= dim or not threads


def test_shapes_of_the_gpu_tests_reach_every_norm():
    forms = {_native.lib().ancha_amd_mx_norm_form(r, d) for r, d in N.SHAPES}
    assert forms == {8 * t + p for _, _, t, p in NORMS}


def test_weights_check_what_they_are_made_of():
    with pytest.raises(ValueError, match="on a GPU"):
        mx.Weight(torch.zeros(2 * 4352, dtype=torch.uint8), 128, 64)
    for k, m in ((0, 64), (64, 0), (-1, 64), (1 << 24, 64)):
        with pytest.raises(ValueError, match="no weight"):
            mx.Weight(torch.zeros(0, dtype=torch.uint8), k, m)
