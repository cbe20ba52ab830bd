"""Refusals of the channel norm's and the matrix optimiser's C entry points and host-side checks (no GPU: every call here ends
before its first launch)."""
import ctypes as C

import numpy as np
import pytest
import torch

from pose_transfer_amd.runtime import lib as L
from pose_transfer_amd.runtime import ops as O

P = 4096          # an aligned address that no refused call reads


def rms(**kw):
    a = dict(x=P, res=None, gamma=P, rows=4, C=64, ldx=64, ldr=64, eps=1e-6, io=0, h=None, y=P * 2, ldy=64, q=None, scales=None, group=0,
             rstd=None)
    a.update(kw)
    return L.load().pg_rms_norm_fwd(a["x"], a["res"], a["gamma"], a["rows"], a["C"], a["ldx"], a["ldr"], a["eps"], a["io"], a["h"], a["y"],
                                    a["ldy"], a["q"], a["scales"], a["group"], a["rstd"], None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(gamma=None), dict(rows=-1), dict(C=0), dict(ldx=63), dict(eps=-1.0), dict(io=1), dict(y=None), dict(res=P, ldr=8),
    dict(ldy=10), dict(q=P), dict(q=P, scales=P, group=48), dict(q=P, scales=P, group=-1), dict(x=P + 2), dict(x=P + 1, io=3), dict(gamma=P + 2),
    dict(C=4096, ldx=4096, ldy=4096, y=P), dict(h=P, ldx=70), dict(y=P, ldx=70), dict(rows=1 << 40, C=4096, ldx=4096, ldy=4096)])
def test_rms_norm_fwd_refuses(bad):
    assert rms(**bad) != 0
    assert L.load().pg_last_error().decode().startswith("pg_rms_norm_fwd")


def test_rms_norm_accepts_no_rows():
    assert rms(rows=0) == 0


def rms_bwd(**kw):
    a = dict(dy=P, lddy=64, dh=None, h=P * 3, rstd=P, gamma=P, rows=4, C=64, io=0, dx=P * 2, dgamma=P, acc=0, ws=None, wsb=0)
    a.update(kw)
    return L.load().pg_rms_norm_bwd(a["dy"], a["lddy"], a["dh"], a["h"], a["rstd"], a["gamma"], a["rows"], a["C"], a["io"], a["dx"], a["dgamma"],
                                    a["acc"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("bad", [
    dict(dy=None), dict(h=None), dict(rstd=None), dict(gamma=None), dict(dx=None), dict(dgamma=None), dict(rows=-1), dict(C=0), dict(lddy=63),
    dict(io=2), dict(dy=P + 2), dict(rows=100000), dict(rows=100000, ws=P, wsb=16), dict(dx=P, lddy=65),
    dict(C=4096, lddy=4096, dx=P, ws=P, wsb=1 << 30)])
def test_rms_norm_bwd_refuses(bad):
    assert rms_bwd(**bad) != 0
    assert L.load().pg_last_error().decode().startswith("pg_rms_norm_bwd")


def orth(**kw):
    a = dict(x=P, xb=0, batch=2, rows=8, cols=16, xs=128, ldx=16, out=P * 2, ob=0, os=128, ldo=16, steps=5, eps=1e-7, ws=P, wsb=1 << 40)
    a.update(kw)
    return L.load().pg_orthogonalise(a["x"], a["xb"], a["batch"], a["rows"], a["cols"], a["xs"], a["ldx"], a["out"], a["ob"], a["os"], a["ldo"],
                                     a["steps"], a["eps"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(batch=-1), dict(rows=-1), dict(cols=-1), dict(ldx=15), dict(ldo=15), dict(os=100), dict(steps=0),
    dict(steps=33), dict(eps=0.0), dict(eps=-1.0), dict(x=P + 2), dict(out=P + 1, ob=1), dict(ws=P + 128), dict(ws=None), dict(wsb=100),
    dict(rows=1 << 17, cols=1 << 17, ldx=1 << 17, ldo=1 << 17, batch=1), dict(rows=1 << 33, batch=1), dict(batch=1 << 31), dict(xs=-1)])
def test_orthogonalise_refuses(bad):
    assert orth(**bad) != 0
    assert L.load().pg_last_error().decode().startswith("pg_orthogonalise")


def test_orthogonalise_empty_and_workspace():
    lib = L.load()
    assert orth(batch=0) == 0 and orth(rows=0) == 0 and orth(cols=0) == 0
    assert lib.pg_orthogonalise_workspace(0, 4, 4) == 0
    assert lib.pg_orthogonalise_workspace(1, 1 << 17, 1 << 17) == -1
    a, b = (lib.pg_orthogonalise_workspace(n, 300, 700) for n in (1, 5))
    assert 0 < a < b < 6 * a


@pytest.mark.parametrize("rows,cols", [(1, (1 << 31) - 1), ((1 << 31) - 1, 1), (1, (1 << 31) - 40), (2, 1 << 30), (1, 1 << 26)])
def test_orthogonalise_refuses_long_thin_matrices(rows, cols):
    """a side near 2^31 rounds up past 32 bits: refused, never wrapped to a small padded size"""
    assert L.load().pg_orthogonalise_workspace(1, rows, cols) == -1
    assert orth(batch=1, rows=rows, cols=cols, ldx=cols, ldo=cols) != 0
    t = table([(0, 1, rows, cols, 0, 1.0)])
    assert L.load().pg_muon_workspace(t.ctypes.data, 1) == -1
    assert muon(entries=[(0, 1, rows, cols, 0, 1.0)], total=1 << 40) != 0


def table(rows):
    return np.array([tuple(r) + (0,) for r in rows], dtype=O.MUON_ENTRY)


GOOD = [(0, 16, 8, 20, 0, 1.0), (2624, 1, 1, 5, 1, 0.0)]


def muon(entries=GOOD, **kw):
    t = table(entries) if entries is not None else None
    a = dict(p=P, g=P * 2, m=P * 3, v=P * 4, entries=t.ctypes.data if t is not None else None, total=1 << 30, n=len(t) if t is not None else 0,
             nesterov=1, steps=5, lr=0.1, momentum=0.9, weight_decay=0.0, grad_scale=1.0, eps=1e-7, beta1=0.5, beta2=0.9, adam_eps=1e-8, step=1,
             workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    return L.load().pg_muon_step(C.byref(L.MuonDesc(**a)), None)


@pytest.mark.parametrize("bad", [
    dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(p=P + 4), dict(g_bf16=P + 2), dict(p_bf16=P + 4), dict(workspace=None),
    dict(workspace=P + 16), dict(workspace_bytes=64), dict(steps=0), dict(steps=40), dict(eps=0.0), dict(total=2600), dict(n=-1), dict(entries=None),
    dict(entries=[(0, 16, 8, 24, 2, 1.0)]), dict(entries=[(0, 0, 8, 24, 0, 1.0)]), dict(entries=[(0, 1, -8, 24, 0, 1.0)]),
    dict(entries=[(0, 1, 8, 0, 1, 1.0)]), dict(entries=[(-64, 1, 8, 24, 0, 1.0)]), dict(entries=[(0, 1, 1 << 16, 1 << 16, 0, 1.0)]),
    dict(entries=[(0, 1 << 20, 1 << 20, 1, 1, 1.0)]), dict(entries=[(0, 1, 8, 24, 0, 1.0), (100, 1, 8, 24, 0, 1.0)]),
    dict(entries=[(1024, 1, 8, 24, 0, 1.0), (0, 1, 8, 24, 0, 1.0)])])
def test_muon_step_refuses(bad):
    bad = dict(bad)
    if "entries" in bad:
        assert muon(entries=bad.pop("entries"), **bad) != 0
    else:
        assert muon(**bad) != 0
    assert L.load().pg_last_error().decode().startswith("pg_muon_step")


def test_muon_step_refuses_sizes_behind_the_address_space():
    """a count or an offset that no arena can have ends in an error, not in an exception of the allocator or a wrapped sum"""
    t = table(GOOD)
    assert L.load().pg_muon_workspace(t.ctypes.data, (1 << 16) + 1) == -1
    assert muon(n=(1 << 31) - 1) != 0
    assert "65536" in L.load().pg_last_error().decode()
    assert muon(entries=[((1 << 63) - 1, 1, 8, 24, 0, 1.0)], total=(1 << 63) - 1) != 0
    assert "ends behind the arena" in L.load().pg_last_error().decode()


def test_muon_tables():
    lib = L.load()
    assert lib.pg_muon_workspace(None, 0) == 0
    t = table([(0, 1, 1 << 16, 1 << 16, 0, 1.0)])
    assert lib.pg_muon_workspace(t.ctypes.data, 1) == -1
    assert O.MUON_ENTRY.itemsize == 32
    assert muon(entries=GOOD[:0]) == 0


def test_wrappers_refuse_on_the_host():
    x, g = torch.zeros(4, 8), torch.ones(8)
    for f in (lambda: O.rms_norm(x, g), lambda: O.rms_norm_q8(x, g), lambda: O.rms_norm_bwd(x, x, torch.ones(4), g),
              lambda: O.orthogonalise(x), lambda: O.orthogonalise(x.half()),
              lambda: O.muon_step(x[0], x[0], x[0], x[0], table(GOOD), lr=0.1), lambda: O.muon_step(x[0], x[0], x[0], x[0], GOOD, lr=0.1)):
        with pytest.raises(ValueError):
            f()


def test_sizes_that_32_bits_do_not_hold():
    """ctypes wraps an argument that its type does not hold, and a row's end plus a turn of the lanes must fit an int"""
    for n in ((1 << 30) + 1, (1 << 32) + 8):
        with pytest.raises(ValueError):
            O._channels(n)
    O._channels(1 << 30)
    n = (1 << 31) - 1
    assert rms(rows=1, C=n, ldx=n, ldy=n) != 0 and "2^30" in L.load().pg_last_error().decode()
    assert rms_bwd(rows=1, C=n, lddy=n, ws=P, wsb=1 << 40) != 0 and "2^30" in L.load().pg_last_error().decode()
    assert rms(rows=(1 << 40) + 1) != 0 and rms_bwd(rows=(1 << 40) + 1, ws=P, wsb=1 << 40) != 0


def test_muon_table_of_the_networks():
    """every element of an arena is in exactly one record; the matrices are the inner blocks' filters"""
    from pose_transfer_amd.runtime import engine as E
    from pose_transfer_amd.utils import synth
    enc, dec = synth.nfilters((256, 256))
    gspec, dspec = synth.generator_spec(18, enc, dec), synth.discriminator_spec(42)
    for spec, order in ((gspec, E.generator_param_order(gspec, len(enc), len(dec))), (dspec, E.discriminator_param_order(dspec))):
        arena = E.ParamArena(spec, order, "cpu")
        t = arena.muon_table()
        end = 0
        for e in t:
            assert end <= e["off"] < end + 64
            assert bool((arena.params[end:int(e["off"])] == 0).all())
            end = int(e["off"]) + int(e["taps"]) * int(e["rows"]) * int(e["cols"])
        assert end <= arena.total < end + 64
        mats = [k for k in arena.keys if arena.is_matrix(k)]
        assert len(mats) == sum(int(e["kind"] == 0) for e in t)
        assert all(k.endswith(".net.1.weight") for k in mats)
        assert sum(arena.numel[k] for k in mats) > 0.97 * sum(arena.numel.values())
        assert O.muon_workspace(t) > 8 * sum(arena.numel[k] for k in mats)


def test_optimizer_option():
    from types import SimpleNamespace
    from pose_transfer_amd.models import pose_gan as G
    from pose_transfer_amd.opts import opts
    o = opts().parse(["--optimizer", "muon", "--muon_momentum", "0.9", "--muon_weight_decay", "0.05"])
    m = G.make_optimizer(None, o)
    assert type(m) is G.FusedMuon and (m.momentum, m.weight_decay, m.lr, m.betas) == (0.9, 0.05, 2e-4, (0.5, 0.999))
    assert type(G.make_optimizer(None, opts().parse([]))) is G.FusedAdam
    assert type(G.make_optimizer(None, SimpleNamespace(learning_rate=1e-3))) is G.FusedAdam
    with pytest.raises(Exception):
        G.make_optimizer(None, SimpleNamespace(learning_rate=1e-3, optimizer="sgd"))
