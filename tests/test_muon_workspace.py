"""The orthogonalised step's workspace: X twice and its lower half, A and B, and no more than 2048 sums of squares a matrix,
which every workgroup that makes a tile of X adds up."""

from __future__ import annotations

import pytest

from flash_maxsim_amd import _lib
from flash_maxsim_amd.flash_maxsim_muon import _Matrix


def padded(n):
    return -(-n // 64) * 64


@pytest.mark.parametrize("rows,cols", [(1, 1), (100, 300), (1024, 4096), (4096, 4096), (4097, 4096), (1 << 14, 1 << 14), (8192, 28672),
                                       (4104, 1 << 20), ((1 << 20) - 24, 4104), (1 << 14, 1 << 20)])
def test_sums_of_squares_are_bounded(rows, cols):
    n, m = sorted((padded(rows), padded(cols)))
    arrays = 3 * 2 * n * m + 2 * 2 * n * n
    chunks = min(2048, -(-rows * cols // 8192))
    got = _lib.load().fmx_muon_workspace_bytes((_Matrix * 1)(_Matrix(None, None, None, None, rows, cols)), 1)
    assert arrays + 8 <= got <= arrays + 8 * chunks + 255
