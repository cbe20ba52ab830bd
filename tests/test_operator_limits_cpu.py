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


def table(rows):
    return np.array([tuple(r) + (0,) for r in rows], dtype=O.MUON_ENTRY)


GOOD = [(0, 16, 8, 20, 0, 1.0), (2624, 1, 1, 5, 1, 0.0)]


def muon(entries=GOOD, **kw):
    t = table(entries)
    a = dict(p=P, g=P * 2, m=P * 3, v=P * 4, entries=t.ctypes.data, total=1 << 30, n=len(t), nesterov=1, steps=5, lr=0.1, momentum=0.9,
             weight_decay=0.0, grad_scale=1.0, eps=1e-7, beta1=0.5, beta2=0.9, adam_eps=1e-8, step=1, workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    return L.load().pg_muon_step(C.byref(L.MuonDesc(**a)), None)


@pytest.mark.parametrize("bad", [dict(step=0), dict(step=-3), dict(step=0, ctr=P), dict(beta1=1.0), dict(beta2=1.0), dict(beta2=-0.1),
                                 dict(beta1=float("nan"))])
def test_muon_step_refuses_corrections_that_divide_by_zero(bad):
    """1 - beta^0 = 0: the Adam records would become infinite or NaN"""
    assert muon(**bad) != 0
    assert "step >= 1 and betas in [0, 1)" in L.load().pg_last_error().decode()


@pytest.mark.parametrize("bad", [dict(ldh=63), dict(ldh=70, dx=P * 3), dict(lddy=63), dict(h=None)])
def test_rms_norm_bwd_ex_refuses(bad):
    a = dict(dy=P, lddy=64, h=P * 3, ldh=64, dx=P * 2)
    a.update(bad)
    assert L.load().pg_rms_norm_bwd_ex(a["dy"], a["lddy"], None, a["h"], a["ldh"], P, P, 4, 64, 0, a["dx"], P, 0, None, 0, None) != 0
    assert L.load().pg_last_error().decode().startswith("pg_rms_norm_bwd")
