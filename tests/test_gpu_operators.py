"""Channel RMS norm and matrix optimiser (runtime/ops.py over include/posegan_hip.h) against plain implementations in 64 bits.

Tolerances.  u = 2^-24 is the rounding of an fp32 operation, EPS the half step of the stored type (bf16 2^-8, fp32 2^-24).
  rms forward:  s is a sum of C squares (at most 32 in sequence, then a tree), a square root and a division, y two more products:
                under 48 u relative, and the store's rounding.
  rms backward: each term of dx carries the same relative error against its own size: 64 u (|w| + |xh| mean|w xh|) s, and the
                stores; dgamma: (rows + 64) u sum|dy xh|, the bound of a sum in any order.
  orthogonal factor: operands of 22 bits and fp32 sums perturb each iterate by at most 2^-20 of its norm; later steps amplify that by at most
                3.4445 each, together under 3.4445^steps 1.5; half of it at least lies along the result (2-norm over all elements).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
NS = (3.4445, -4.7750, 2.0315)


def ops():
    from pose_transfer_amd.runtime import ops as O
    return O


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ------------------------------------------------------------------------------------------------ rms norm
def rms_ref(x, gamma, res, eps):
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    d = h.double()
    s = 1.0 / torch.sqrt((d * d).mean(1) + eps)
    return h, s, d * s[:, None] * gamma.double()


ROWS_C = [(1, 1), (1, 512), (3, 7), (2, 8), (5, 31), (17, 64), (33, 65), (9, 128), (130, 189), (7, 513), (4, 1024), (3, 1536), (2, 2048),
          (2, 2049), (1, 5003)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", ROWS_C)
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm_forward(dtype, rows, C, res):
    x = rnd(1, rows, C + 3, dtype=dtype)[:, 1:C + 1]          # strided rows, odd alignment
    r = rnd(2, rows, C, dtype=dtype) if res else None
    gamma = rnd(3, C) + 1.0
    y, h, rstd = ops().rms_norm(x, gamma, r, eps=1e-5)
    hr, sr, yr = rms_ref(x, gamma, r, 1e-5)
    assert torch.equal(h, hr)
    assert bool(((rstd.double() - sr).abs() <= 48 * U * sr).all())
    assert bool(((y.double() - yr).abs() <= (EPS[dtype] * 1.01 + 48 * U) * yr.abs()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", ROWS_C)
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
def test_rms_norm_q8(dtype, rows, C, group):
    x, r = rnd(4, rows, C, dtype=dtype), rnd(5, rows, C, dtype=dtype)
    if C > 300:
        x[0, 256:512] = 0                                     # a group of zeros
        r[0, 256:512] = 0
    gamma = rnd(6, C) + 1.0
    q, scale, h, rstd = ops().rms_norm_q8(x, gamma, r, group=group)
    hr, sr, yr = rms_ref(x, gamma, r, 1e-6)
    assert torch.equal(h, hr)
    g = group or C
    n = -(-C // g)
    assert tuple(scale.shape) == (rows, n)
    yp = torch.nn.functional.pad(yr, (0, n * g - C)).view(rows, n, g)
    top = yp.abs().amax(2)
    want = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    assert bool(((scale.double() - want).abs() <= 64 * U * want).all())
    back = q.float().double() * scale.double().repeat_interleave(g, 1)[:, :C]
    step = want.repeat_interleave(g, 1)[:, :C]
    # half a step of e4m3: 2^-4 relative, 2^-10 below its smallest normal
    assert bool(((back - yr).abs() <= (2.0 ** -4 + 128 * U) * yr.abs() + 2.0 ** -10 * step).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", ROWS_C + [(700, 40), (3000, 129), (300, 2048)])
@pytest.mark.parametrize("dh", [False, True])
def test_rms_norm_backward(dtype, rows, C, dh):
    h = rnd(7, rows, C, dtype=dtype)
    dy = rnd(8, rows, C + 5, dtype=dtype)[:, 3:C + 3]
    d = rnd(9, rows, C, dtype=dtype) if dh else None
    gamma = rnd(10, C) + 1.0
    s = 1.0 / torch.sqrt(h.double().square().mean(1) + 1e-6)
    dx, dgamma = ops().rms_norm_bwd(dy, h, s.float(), gamma, dh=d)
    s = s.float().double()[:, None]
    xh = h.double() * s
    w = dy.double() * gamma.double()
    ref = s * (w - xh * (w * xh).mean(1, keepdim=True))
    size = s * (w.abs() + xh.abs() * (w * xh).abs().mean(1, keepdim=True))
    if dh:
        ref, size = ref + d.double(), size + d.double().abs()
    assert bool(((dx.double() - ref).abs() <= EPS[dtype] * 1.01 * ref.abs() + 64 * U * size).all())
    t = dy.double() * xh
    assert bool(((dgamma.double() - t.sum(0)).abs() <= (rows + 64) * U * t.abs().sum(0)).all())


def test_rms_norm_gradient_against_differences():
    """the gradients of sum(wy y) + sum(wh h) against central differences of the 64-bit definition"""
    rows, C = 5, 37
    x, r, gamma = rnd(11, rows, C), rnd(12, rows, C), rnd(13, C) + 1.0
    wy, wh = rnd(14, rows, C), rnd(15, rows, C)
    y, h, rstd = ops().rms_norm(x, gamma, r)
    dx, dgamma = ops().rms_norm_bwd(wy, h, rstd, gamma, dh=wh)

    def f(xx, gg):
        hh = xx + r.double()
        yy = hh / torch.sqrt((hh * hh).mean(1, keepdim=True) + 1e-6) * gg
        return float((wy.double() * yy).sum() + (wh.double() * hh).sum())
    t = 1e-5
    for i, j in ((0, 0), (2, 17), (4, 36)):
        e = torch.zeros(rows, C, dtype=torch.float64, device="cuda")
        e[i, j] = t
        num = (f(x.double() + e, gamma.double()) - f(x.double() - e, gamma.double())) / (2 * t)
        assert abs(num - float(dx[i, j])) < 2e-4          # differences: O(t^2) + 1e-16 * 200 / t; dx: a few u of terms of size 5
        e = torch.zeros(C, dtype=torch.float64, device="cuda")
        e[j] = t
        num = (f(x.double(), gamma.double() + e) - f(x.double(), gamma.double() - e)) / (2 * t)
        assert abs(num - float(dgamma[j])) < 2e-4


def test_rms_norm_special_values():
    x = rnd(16, 6, 96)
    x[1] = 0                                                  # an empty row: rstd = eps^-1/2, y = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    gamma = torch.ones(96, device="cuda")
    y, h, rstd = ops().rms_norm(x, gamma, eps=1e-6)
    assert torch.equal(y[1], torch.zeros(96, device="cuda")) and abs(float(rstd[1]) - 1e3) < 0.1
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3, 7])) and float(y[3, :7].abs().max()) == 0
    ok = [0, 1, 4, 5]
    assert bool(torch.isfinite(y[ok]).all())
    q, scale, _, _ = ops().rms_norm_q8(x, gamma, group=32)
    assert bool((scale[1] == 1).all()) and float(q[1].float().abs().max()) == 0
    q0, scale0, _, _ = ops().rms_norm_q8(x[ok].contiguous(), gamma, group=32)
    assert torch.equal(q[ok].view(torch.uint8), q0.view(torch.uint8)) and torch.equal(scale[ok], scale0)


def test_rms_norm_more_rows_than_one_launch_holds():
    """2^28 rows of one channel fill a launch of eight lanes each: the rows behind them too"""
    O = ops()
    n = (1 << 28) + 77
    x = torch.arange(n, device="cuda", dtype=torch.int32).remainder_(7).to(torch.bfloat16).add_(1).view(n, 1)
    gamma = torch.full((1,), 0.5, device="cuda")
    y, _, rstd = O.rms_norm(x, gamma)
    # h rstd gamma = 0.5 / sqrt(1 + eps / h^2): 0.5 in bf16
    assert bool((y == 0.5).all())
    assert float((rstd * x[:, 0].float() - 1).abs().max()) < 1e-6
    del y
    q, scale, _, _ = O.rms_norm_q8(x, gamma)
    assert bool((q.view(torch.uint8) == q.view(torch.uint8)[0, 0]).all())
    assert float((scale * q[0, 0].float() - 0.5).abs().max()) < 1e-6          # 1e-6 / 2 (eps) and three roundings of 2^-25
    del x, q, scale, rstd
    n, c = (1 << 23) + 3, 2049                             # a workgroup per row: 34 GB a tensor
    h = torch.ones(n, c, dtype=torch.bfloat16, device="cuda")
    rstd = torch.ones(n, device="cuda")
    g = torch.ones(c, device="cuda")
    h[-1] = 2.0
    dx, dgamma = O.rms_norm_bwd(h, h, rstd, g)              # w = xh: dx = h - h mean(h^2)
    assert bool((dx[:-1] == 0).all()) and bool((dx[-1] == -6).all())
    del dx
    assert float((dgamma - (n + 3)).abs().max()) <= 2.0 ** -24 * (n + 3)
    h[-1] = 3.0
    y, _, r = O.rms_norm(h, g, eps=0.0)
    assert bool((y == 1).all()) and float((r[-1] - 1 / 3).abs()) < 1e-7
    del y, h
    torch.cuda.empty_cache()


def test_rms_norm_empty_and_other_stream():
    O = ops()
    e = torch.empty(0, 64, device="cuda")
    gamma = torch.ones(64, device="cuda")
    y, h, rstd = O.rms_norm(e, gamma)
    assert y.shape == (0, 64) and rstd.shape == (0,)
    dx, dg = O.rms_norm_bwd(e, e, rstd, gamma)
    assert dx.shape == (0, 64) and float(dg.abs().max()) == 0
    x = rnd(17, 300, 64)
    want = O.rms_norm(x, gamma)[0]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = O.rms_norm(x, gamma)[0]
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ orthogonalisation
def ortho_ref(x, steps=5, eps=1e-7):
    d = x.double()
    z = d if d.shape[0] <= d.shape[1] else d.t()
    z = z / (z.norm() + eps)
    for _ in range(steps):
        A = z @ z.t().contiguous()
        z = NS[0] * z + (NS[1] * A + NS[2] * (A @ A)) @ z
    return z if d.shape[0] <= d.shape[1] else z.t()


def close(got, ref, steps=5):
    tol = EPS[got.dtype] + 1.5 * NS[0] ** steps * 2.0 ** -20
    err = float((got.double() - ref).norm() / ref.norm())
    assert err <= tol, (err, tol)


SHAPES = [(1, 1, 1), (1, 1, 7), (1, 7, 1), (2, 2, 2), (3, 64, 64), (2, 65, 63), (1, 128, 300), (2, 300, 130), (1, 257, 1025), (1, 33, 4099),
          (1, 4099, 33), (5, 16, 200), (1, 192, 9216), (1, 640, 700), (3, 50, 384), (2, 384, 64), (2, 64, 385), (2, 100, 2000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalise(dtype, shape):
    x = rnd(20, *shape, dtype=dtype, scale=1e-3)
    for out_dtype in (torch.float32, torch.bfloat16):
        o = ops().orthogonalise(x, out_dtype=out_dtype)
        assert o.dtype == out_dtype and o.shape == x.shape
        for b in range(shape[0]):
            close(o[b], ortho_ref(x[b]))


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_orthogonalise_steps(steps):
    x = rnd(21, 90, 260)
    # an input whose singular values are alike: the amplification of seven steps has nothing to work on
    x = torch.linalg.qr(x.double().t())[0].t().float().contiguous() + 0.01 * x
    close(ops().orthogonalise(x, steps=steps), ortho_ref(x, steps), min(steps, 5))


def test_orthogonalise_singular_values_and_spectra():
    g = torch.Generator().manual_seed(3)
    u = torch.linalg.qr(torch.randn(150, 150, generator=g, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(700, 150, generator=g, dtype=torch.float64))[0]
    for power in (0.0, 0.5, 1.0, 2.0):
        x = ((u * torch.arange(1, 151).double() ** -power) @ v.t()).float().cuda()
        o = ops().orthogonalise(x)
        close(o, ortho_ref(x))
        if power < 1:
            s = torch.linalg.svdvals(o.double().cpu())
            assert 0.6 < float(s.min()) and float(s.max()) < 1.25


def test_orthogonalise_large_batches():
    """a batch that does not fit one launch (lanes of the one-launch form) or one workspace goes in pieces: every matrix gets what it
    gets by itself, a piece's last one and the next one's first among them"""
    from pose_transfer_amd.runtime import lib as L
    O = ops()
    n = (1 << 23) + 5
    x = rnd(46, n, 2, 2)
    out = O.orthogonalise(x)
    for sl in (slice(0, 3), slice((1 << 22) - 2, (1 << 22) + 2), slice((1 << 23) - 2, n)):
        assert torch.equal(out[sl], O.orthogonalise(x[sl])), sl
    n = 12000
    assert L.load().pg_orthogonalise_workspace(n, 1, 385) <= 1 << 31 < n * (2 * 2 * 448 * 72 * 2)
    x = rnd(47, n, 1, 385, dtype=torch.bfloat16)
    out = O.orthogonalise(x, out_dtype=torch.float32).double()
    ref = x.double()
    ref = ref / (ref.norm(dim=2, keepdim=True) + 1e-7)
    for _ in range(5):                                        # one row: A = |x|^2
        a = (ref * ref).sum(2, keepdim=True)
        ref = (NS[0] + NS[1] * a + NS[2] * a * a) * ref
    assert float(((out - ref).norm(dim=2) / ref.norm(dim=2)).max()) <= 1.5 * NS[0] ** 5 * 2.0 ** -20


def test_orthogonalise_scales_strides_and_special_values():
    O = ops()
    x = rnd(22, 4, 70, 210)
    base = O.orthogonalise(x)
    for f in (2.0 ** -30, 2.0 ** 40):                         # powers of two: the planes are the same
        # eps weighs differently: against its own definition
        close(O.orthogonalise(x[0] * f), ortho_ref(x[0] * f))
    assert torch.equal(O.orthogonalise(x * 2.0 ** 20, eps=1e-30), O.orthogonalise(x, eps=1e-30))
    wide = torch.zeros(4, 75, 230, device="cuda")
    wide[:, 2:72, 3:213] = x
    assert torch.equal(O.orthogonalise(wide[:, 2:72, 3:213]), base)
    assert torch.equal(O.orthogonalise(x[:1].expand(3, 70, 210)), base[:1].expand(3, 70, 210))
    assert torch.equal(O.orthogonalise(x.transpose(1, 2)).transpose(1, 2), O.orthogonalise(x.transpose(1, 2).contiguous()).transpose(1, 2))
    assert torch.equal(O.orthogonalise(x[1]), base[1])        # one alone and one of a batch: the same sums
    y = x.clone()
    y[0, 3, 5] = float("nan")
    y[1, 0, 0] = float("inf")
    y[2] = 0
    o = O.orthogonalise(y)
    assert bool(torch.isnan(o[0]).all()) and bool(torch.isnan(o[1]).all())
    assert float(o[2].abs().max()) == 0
    assert torch.equal(o[3], base[3])
    one = torch.zeros(40, 100, device="cuda")
    one[7, 9] = 5.0                                           # rank one, largest over rms as far as it goes
    close(O.orthogonalise(one), ortho_ref(one))
    assert O.orthogonalise(torch.empty(0, 3, 4, device="cuda")).shape == (0, 3, 4)
    assert O.orthogonalise(torch.empty(3, 0, device="cuda")).shape == (3, 0)


# ------------------------------------------------------------------------------------------------ Muon step
def table_of(parts):
    O = ops()
    rec, off = [], 0
    for p in parts:
        if len(p) == 1:
            n, r = p[0], (off, 1, 1, p[0], 1, 0.0, 0)
        else:
            n, r = p[0] * p[1] * p[2], (off,) + tuple(p) + (0, 0.2 * math.sqrt(max(p[1], p[0] * p[2])), 0)
        rec.append(r)
        off += (n + 63) // 64 * 64
    return np.array(rec, dtype=O.MUON_ENTRY), off


def muon_ref(p, g, m, v, table, lr, mu, nesterov, wd, b1, b2, eps, step):
    p, g, m, v = (t.double().clone() for t in (p, g, m, v))
    # the kernel holds mu, 1 - mu and the other coefficients in fp32
    f = lambda c: float(np.float32(c))
    for e in table:
        taps, rows, cols = int(e["taps"]), int(e["rows"]), int(e["cols"])
        at = slice(int(e["off"]), int(e["off"]) + taps * rows * cols)
        if e["kind"] == 0:
            m[at] = f(mu) * m[at] + (1 - f(mu)) * g[at]
            u = (1 - f(mu)) * g[at] + f(mu) * m[at] if nesterov else m[at]
            x = u.view(taps, rows, cols).permute(1, 0, 2).reshape(rows, taps * cols)
            o = ortho_ref(x).reshape(rows, taps, cols).permute(1, 0, 2).reshape(-1)
            p[at] = p[at] * (1 - f(lr) * f(wd)) - f(lr) * float(e["scale"]) * o
        else:
            m[at] = f(b1) * m[at] + (1 - f(b1)) * g[at]
            v[at] = f(b2) * v[at] + (1 - f(b2)) * g[at] * g[at]
            p[at] = p[at] - lr / (1 - b1 ** step) * m[at] / (v[at].sqrt() / math.sqrt(1 - b2 ** step) + eps)
    return p, m, v


PARTS = [[(1, 1, 1)], [(16, 64, 48)], [(65,), (9, 30, 21), (3,), (16, 130, 70), (1,)], [(1, 300, 20), (4, 50, 5), (64,)],
         [(5000,)], [(16, 128, 64), (16, 256, 128), (1,), (1,), (9, 3, 17), (9, 17, 3), (1, 2, 5000)]]


@pytest.mark.parametrize("parts", PARTS)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("gbf", [False, True])
def test_muon_step(parts, nesterov, gbf):
    table, total = table_of(parts)
    p, g, m, v = rnd(30, total, scale=0.05), rnd(31, total, scale=1e-3), rnd(32, total, scale=1e-3), rnd(33, total).square() * 1e-6
    if gbf:
        g = g.bfloat16()
    p0, m0, v0 = p.clone(), m.clone(), v.clone()
    pb = torch.full((total,), 7.0, dtype=torch.bfloat16, device="cuda")
    ops().muon_step(p, g, m, v, table, lr=2e-3, momentum=0.95, nesterov=nesterov, weight_decay=0.1, betas=(0.5, 0.999), eps=1e-8, step=4,
                    p_bf16=pb)
    pr, mr, vr = muon_ref(p0, g, m0, v0, table, 2e-3, 0.95, nesterov, 0.1, 0.5, 0.999, 1e-8, 4)
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for e in table:
        n = int(e["taps"]) * int(e["rows"]) * int(e["cols"])
        at = slice(int(e["off"]), int(e["off"]) + n)
        used[at] = True
        a, b = p[at].double() - p0[at].double(), pr[at] - p0[at].double()
        # the update against its own size, and the last rounding of p
        tol = 1.5 * NS[0] ** 5 * 2.0 ** -20 + 16 * U
        assert float((a - b).norm()) <= tol * float(b.norm()) + 2 * U * float(p0[at].double().norm()) + 2 * U * float(pr[at].norm())
    assert bool(((m.double() - mr).abs() <= 4 * U * (m0.double().abs() + g.double().abs())).all())
    assert bool(((v.double() - vr).abs() <= 8 * U * vr.abs()).all())
    assert torch.equal(p[~used], p0[~used]) and torch.equal(m[~used], m0[~used]) and bool((pb[~used] == 7).all())
    assert torch.equal(pb[used], p[used].bfloat16())


def test_muon_step_repeats_bit_for_bit_and_counts_on_the_device():
    table, total = table_of(PARTS[2])
    outs = []
    for k in range(3):
        p, g, m, v = rnd(40, total, scale=0.05), rnd(41, total), rnd(42, total), rnd(43, total).square()
        ctr = torch.tensor([3], dtype=torch.int64, device="cuda") if k == 2 else None
        ops().muon_step(p, g, m, v, table, lr=1e-3, step=2 if k == 2 else 5, ctr=ctr, grad_scale=0.5)
        outs.append((p, m, v))
    for k in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(outs[0], outs[k]))


def test_operators_in_a_captured_graph():
    """the three operators as a training step uses them, captured once and replayed between eager calls"""
    O = ops()
    table, total = table_of([(1, 96, 160), (160,)])
    gamma = torch.ones(160, device="cuda")
    x, r, dy = rnd(50, 40, 160), rnd(51, 40, 160), rnd(52, 40, 160)

    def step(p, m, v):
        y, h, rstd = O.rms_norm(x, gamma, r)
        dx, dgamma = O.rms_norm_bwd(dy, h, rstd, gamma, dh=r)
        g = torch.zeros(total, device="cuda")
        g[:96 * 160] = torch.matmul(dy[:, :96].t().contiguous(), y).reshape(-1)
        g[table[1]["off"]:table[1]["off"] + 160] = dgamma
        O.muon_step(p, g, m, v, table, lr=1e-2, step=1)
        o = O.orthogonalise(p[:96 * 160].view(96, 160))
        return dx, o

    def fresh():
        return rnd(53, total), torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    e = fresh()
    want = []
    for _ in range(4):
        dx, o = step(*e)
        want.append((dx.clone(), o.clone(), e[0].clone()))
    s = fresh()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(*[t.clone() for t in s])
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, o = step(*s)
    for k in range(4):
        graph.replay()
        junk = O.orthogonalise(rnd(60 + k, 200, 300))         # the program's own work between replays
        torch.cuda.synchronize()
        assert torch.equal(dx, want[k][0]) and torch.equal(o, want[k][1]) and torch.equal(s[0], want[k][2]), k
        assert bool(torch.isfinite(junk).all())


def test_two_streams_at_once():
    """calls on two streams side by side, each with workspaces of its own: what each gets alone"""
    O = ops()
    a, b = rnd(90, 3, 200, 900), rnd(91, 2, 130, 2000, dtype=torch.bfloat16)
    dy, h = rnd(92, 5000, 129), rnd(93, 5000, 129)
    g, rstd = rnd(94, 129), torch.ones(5000, device="cuda")
    want_a, want_b, want_n = O.orthogonalise(a), O.orthogonalise(b), O.rms_norm_bwd(dy, h, rstd, g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(8):
        with torch.cuda.stream(streams[0]):
            got.append((O.orthogonalise(a), want_a))
            got.append((O.rms_norm_bwd(dy, h, rstd, g)[1], want_n[1]))
        with torch.cuda.stream(streams[1]):
            got.append((O.rms_norm_bwd(dy, h, rstd, g)[0], want_n[0]))
            got.append((O.orthogonalise(b), want_b))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ module and trainer
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rms_norm_module(dtype):
    from pose_transfer_amd.models.networks import RMSNorm
    mod = RMSNorm(48)
    with torch.no_grad():
        mod.weight.copy_(rnd(70, 48) + 1.0)
    x, r = rnd(71, 2, 5, 3, 48, dtype=dtype).requires_grad_(), rnd(72, 2, 5, 3, 48, dtype=dtype).requires_grad_()
    wy, wh = rnd(73, 2, 5, 3, 48, dtype=dtype), rnd(74, 2, 5, 3, 48, dtype=dtype)
    y, h = mod(x, r)
    ((y * wy).sum() + (h * wh).sum()).backward()
    xd, rd = x.detach().double().requires_grad_(), r.detach().double().requires_grad_()
    gd = mod.weight.detach().double().requires_grad_()
    hd = xd + rd
    hd = hd + (h.detach().double() - hd).detach()             # the stored sum; its gradient is the sum's
    yd = hd / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-6) * gd
    ((yd * wy.double()).sum() + (hd * wh.double()).sum()).backward()
    # dx: a rounding of its own size, and terms of size |w| + |xh| mean|w xh| <= 60 in 64 u
    assert bool(((x.grad.double() - xd.grad).abs() <= EPS[dtype] * 1.01 * xd.grad.abs() + 64 * U * 60).all())
    assert torch.equal(x.grad, r.grad)
    assert bool(((mod.weight.grad.double() - gd.grad).abs() <= 94 * U * (wy.double() * yd.detach() / gd.detach()).abs().sum((0, 1, 2))).all())
    y = mod(x.detach().requires_grad_())
    assert y.shape == x.shape and y.grad_fn is not None
    (only_h,) = torch.autograd.grad(mod(x, r)[1].sum(), x)
    assert torch.equal(only_h, torch.ones_like(x))


def test_rms_norm_module_layouts_and_refusals():
    """expanded gradients, channels-first inputs and broadcast residuals, as autograd and other layers hand them over"""
    from pose_transfer_amd.models.networks import RMSNorm
    mod = RMSNorm(24)
    x = rnd(75, 6, 24).requires_grad_()
    mod(x).sum().backward()                                   # the gradient is one expanded element
    want, gw = torch.autograd.grad(mod(x), (x, mod.weight), torch.ones(6, 24, device="cuda"))
    assert torch.equal(x.grad, want) and torch.equal(mod.weight.grad, gw)
    xt = rnd(76, 24, 6).requires_grad_()                      # channels first: a transposed view
    wy = rnd(77, 24, 6)
    (mod(xt.t()) * wy.t()).sum().backward()
    xc = xt.detach().t().contiguous().requires_grad_()
    (mod(xc) * wy.t().contiguous()).sum().backward()
    assert torch.equal(xt.grad.t(), xc.grad)
    r = rnd(78, 1, 24).requires_grad_()                       # one residual row for all
    y, h = mod(x.detach(), r.expand(6, 24))
    (y * h).sum().backward()
    rc = r.detach().repeat(6, 1).requires_grad_()
    y, h = mod(x.detach(), rc)
    (y * h).sum().backward()
    assert torch.equal(r.grad, rc.grad.sum(0, keepdim=True))
    s = rnd(79, 6, 24).requires_grad_()                       # both inputs the same tensor: twice the gradient
    y, h = mod(s, s)
    (y.sum() + (2 * h).sum()).backward()
    s2, s3 = s.detach().clone().requires_grad_(), s.detach().clone().requires_grad_()
    y, h = mod(s2, s3)
    (y.sum() + (2 * h).sum()).backward()
    assert torch.equal(s.grad, s2.grad + s3.grad) and s2.grad.data_ptr() != s3.grad.data_ptr()
    with pytest.raises(ValueError):
        mod(x, torch.zeros(12, 12, device="cuda"))
    with pytest.raises(ValueError):
        mod(rnd(80, 2, 3, 24), rnd(81, 3, 2, 24))
    (g,) = torch.autograd.grad(mod(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def trainer(optimizer, precision=0, n=2, size=64):
    from types import SimpleNamespace
    from pose_transfer_amd.models.pose_gan import DeformablePose_GAN
    from pose_transfer_amd.runtime import engine as E
    from pose_transfer_amd.utils import synth
    E.PRECISION = precision
    opt = SimpleNamespace(image_size=(size, size), use_input_pose=True, pose_dim=18, batch_size=n, num_stacks=4, gen_type="baseline",
                          dataset="fasion", warp_skip="mask", learning_rate=2e-4, content_loss_layer="none", nn_loss_area_size=1,
                          gan_penalty_weight=1.0, l1_penalty_weight=100.0, optimizer=optimizer, muon_momentum=0.9, muon_weight_decay=0.01)
    model = DeformablePose_GAN(opt, device="cuda:0")
    b = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in synth.batch(1, "muon/A", n, 18, size, size)]
    return model, vars(opt), b


def test_trainer_with_muon_against_the_definition():
    """one dis_update and one gen_update: the arenas after each step against the 64-bit step on the arena's own gradients"""
    model, od, b = trainer("muon")
    for arena, run in ((model.disc.arena, lambda: model.dis_update(b[0], b[1], {"warps": b[2], "masks": b[3]}, b[0], b[1], od)),
                       (model.gen.arena, lambda: model.gen_update(b[0], b[1], {"warps": b[2], "masks": b[3]}, od))):
        for step in (1, 2):
            p0, m0, v0 = arena.params.clone(), arena.m.clone(), arena.v.clone()
            losses = run()
            assert losses is not None and arena.step == step
            table = arena.muon_table()
            assert sum(1 for e in table if e["kind"] == 0) == sum(arena.is_matrix(k) for k in arena.keys) >= 3
            pr, mr, vr = muon_ref(p0, arena.grads, m0, v0, table, 2e-4, 0.9, True, 0.01, 0.5, 0.999, 1e-8, step)
            for e in table:
                at = slice(int(e["off"]), int(e["off"]) + int(e["taps"]) * int(e["rows"]) * int(e["cols"]))
                a, r = arena.params[at].double() - p0[at].double(), pr[at] - p0[at].double()
                tol = (1.5 * NS[0] ** 5 * 2.0 ** -20 if e["kind"] == 0 else 0.0) + 64 * U
                assert float((a - r).norm()) <= tol * float(r.norm()) + 2 * U * float(pr[at].norm()) + 2 * U * float(p0[at].norm())
            assert bool(((arena.m.double() - mr).abs() <= 4 * U * (m0.double().abs() + arena.grads.double().abs())).all())
    sd = model.gen.state_dict()
    assert all(bool(torch.isfinite(v).all()) for v in sd.values())


def test_trainer_with_muon_bf16_weights_follow():
    model, od, b = trainer("muon", precision=3)
    from pose_transfer_amd.runtime import engine as E
    try:
        model.dis_update(b[0], b[1], {"warps": b[2], "masks": b[3]}, b[0], b[1], od)
        model.gen_update(b[0], b[1], {"warps": b[2], "masks": b[3]}, od)
        for arena in (model.disc.arena, model.gen.arena):
            assert arena.bf16_version == arena.version()
            for k in arena.keys:
                at = slice(arena.off[k], arena.off[k] + arena.numel[k])
                assert torch.equal(arena.params_bf16[at], arena.params[at].bfloat16())
    finally:
        E.PRECISION = 0


def test_trainer_with_muon_replayed_from_a_tape():
    """recorded launches of the Muon step against the eager loop: same batches, same dropout masks, three iterations"""
    from pose_transfer_amd.runtime.tape import TapedIteration
    from pose_transfer_amd.utils import synth
    runs = []
    for taped in (False, True):
        model, od, b = trainer("muon")
        drop = [m.cuda() for m in (torch.from_numpy(np.ascontiguousarray(a)) for a in synth.dropout_masks(1, "muon/d", 2))]
        b = [b[0], b[1], b[2].float().contiguous(), b[3]]
        if taped:
            t = TapedIteration(model, [b, b, b], dict(od), warmup=1, drop_masks=(drop, drop))     # one eager, one recorded
            t.replay()
            t.close()
        else:
            for _ in range(3):
                o = {"warps": b[2], "masks": b[3], "drop_masks": drop}
                model.dis_update(b[0], b[1], o, b[0], b[1], dict(od, lazy_losses=True))
                model.gen_update(b[0], b[1], o, dict(od, lazy_losses=True))
        torch.cuda.synchronize()
        assert model.gen.arena.step == 3
        runs.append((model.gen.arena.params.clone(), model.disc.arena.params.clone()))
    for a, c in zip(*runs):
        # the trainer's own gradients come from float atomics: equal up to their order, magnified by Adam's and Muon's scaling
        assert float((a - c).norm() / c.norm()) < 1e-2


def test_residual_block_step_uses_all_of_them():
    """norm with the residual -> product -> its gradients -> Muon step, twice, against 64 bits"""
    O = ops()
    rows, C = 192, 64
    x, r, t = rnd(80, rows, C), rnd(81, rows, C), rnd(82, rows, C)
    table, total = table_of([(1, C, C), (C,)])
    gain = slice(int(table[1]["off"]), int(table[1]["off"]) + C)
    p, m, v = rnd(83, total, scale=0.1), torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    p[gain] = 1.0
    pd, md, vd = p.double(), m.double(), v.double()
    for step in (1, 2):
        w = p[:C * C].view(C, C)
        y, h, rstd = O.rms_norm(x, p[gain].contiguous(), r)
        err = y @ w.t() + h - t
        g = torch.zeros(total, device="cuda")
        g[:C * C] = (err.t().contiguous() @ y).reshape(-1)
        dx, g[gain] = O.rms_norm_bwd(err @ w, h, rstd, p[gain].contiguous(), dh=err)
        O.muon_step(p, g, m, v, table, lr=1e-2, step=step)
        # the same in 64 bits with autograd
        wd, gd, xd = pd[:C * C].view(C, C).clone().requires_grad_(), pd[gain].clone().requires_grad_(), x.double().requires_grad_()
        hd = xd + r.double()
        yd = hd / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6) * gd
        loss = 0.5 * (yd @ wd.t() + hd - t.double()).square().sum()
        loss.backward()
        assert float((dx.double() - xd.grad).norm() / xd.grad.norm()) < 1e-5        # fp32 products of 64 terms: about 8 u of the size
        gr = torch.zeros(total, dtype=torch.float64, device="cuda")
        gr[:C * C], gr[gain] = wd.grad.reshape(-1), gd.grad
        pd, md, vd = muon_ref(pd, gr, md, vd, table, 1e-2, 0.95, True, 0.0, 0.5, 0.999, 1e-8, step)
        for at in (slice(0, C * C), gain):
            assert float((p[at].double() - pd[at]).norm() / pd[at].norm()) < 1e-4
