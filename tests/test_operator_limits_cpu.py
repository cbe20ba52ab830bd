"""Limits of the channel norm and the matrix optimiser that show on the host: workspace sizes, refusals (no GPU: every call here ends before
its first launch)."""
import ctypes as C

import numpy as np
import pytest
import torch

from pose_transfer_amd.runtime import lib as L
from pose_transfer_amd.runtime import ops as O

P = 4096          # an aligned address that no refused call reads


def up(a, b):
    return -(-a // b) * b


def planes(short, long_):
    """bytes of a matrix's planes, chain matrices and Gram slices (one 128 x 128 tile of rows: a short side of at most 128)"""
    mp, np_ = up(short, 64), up(long_, 64)
    ks = max(1, min(512, np_ // 256))
    kc = up(-(-np_ // ks), 32)
    return 8 * np_ * (mp + 8) + 20 * mp * (mp + 8) + 4 * 128 * 128 * -(-np_ // kc)


@pytest.mark.parametrize("rows,cols", [(65, 1 << 22), ((1 << 25) - 64, 1), (1 << 22, 65), (128, 1 << 20), (100, 3000)])
def test_partial_sums_of_squares_are_bounded(rows, cols):
    """every workgroup that splits a matrix into planes joins all of its partial sums: 1024 at most, whatever the matrix"""
    most = planes(*sorted((rows, cols))) + 1024 * 16 + 6 * 1024            # and table, units, rounding to 256 bytes
    assert L.load().pg_orthogonalise_workspace(1, rows, cols) <= most
    t = np.array([(0, 1, rows, cols, 0, 1.0, 0)], dtype=O.MUON_ENTRY)
    assert L.load().pg_muon_workspace(t.ctypes.data, 1) <= most
