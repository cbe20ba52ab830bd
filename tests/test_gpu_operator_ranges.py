"""Range and edge tests of the channel norm and the matrix optimiser (runtime/ops.py) beside tests/test_gpu_operators.py, against plain
implementations in 64 bits.

Tolerances.  U = 2^-24, EPS the half step of the stored type.
  orthogonal factor, inputs whose long side is at least four times the short one: a Gaussian's singular values then lie within a factor
      (1 + 1/2) / (1 - 1/2) = 3 of each other.  A step has four products of 22-bit operands, each within 2^-21 of its size; twenty of them,
      magnified by at most that factor: BASE = 20 * 2^-21 * 3 = 2.9e-5.  (Operands of 11 bits, one of the two fp16 values lost, are
      ten times outside.)
  rows much smaller than the others: the m x m factor P of a stage is off by an absolute 2^-30 at most (G by 2^-40, Q by 4.8 times that
      and 2^-39 of its own, three of them multiplied: 36 times, then P's own 2^-35 twice), so a row by 2^-30 sqrt(m) |X|_2, |X|_2 <= 1; the
      row itself, r of the others, grows from r / sqrt(m) to 41 times that: relative 2^-30 m / (41 r).
  columns of the long side (n of them) much smaller than the others: the planes between stages hold 2^15 X to an absolute 2^-25, so a
      column is off by 2^-40 sqrt(m); its own size is at least 0.3 r sqrt(m / n) (0.3: a singular value after the first stage)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
NS = (3.4445, -4.7750, 2.0315)
BASE = 20 * 2.0 ** -21 * 3


def ops():
    from pose_transfer_amd.runtime import ops as O
    return O


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def ortho_ref(x, steps=5, eps=1e-7):
    """one matrix or a batch, in 64 bits, products of batches one by one"""
    if x.dim() == 3:
        return torch.stack([ortho_ref(m, steps, eps) for m in x])
    z = x.double() if x.shape[0] <= x.shape[1] else x.double().t()
    z = z / (z.norm() + eps)
    for _ in range(steps):
        A = z @ z.t().contiguous()
        z = NS[0] * z + (NS[1] * A + NS[2] * (A @ A)) @ z
    return z if x.shape[0] <= x.shape[1] else z.t()


# the one-launch form, both one-workgroup chains, chain tiles of 32 (few matrices) and of 64 (many), wide and tall
ORTHO = [(1, 40, 200), (3, 64, 300), (1, 64, 900), (2, 900, 64), (1, 128, 1152), (2, 1152, 100), (1, 300, 1300), (1, 1300, 300), (12, 300, 1300),
         (12, 1300, 300), (1, 512, 2500), (6, 200, 900)]


@pytest.mark.parametrize("shape", ORTHO)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalise_keeps_small_rows(shape, dtype):
    """rows (of the short side) 1e-3 to 1e-7 of the others: each against its own size"""
    x = rnd(1, *shape)
    tall = shape[1] > shape[2]
    short = min(shape[1:])
    size = torch.ones(short, device="cuda")
    at = [0, 7, 17, 23, 38]
    for i, r in zip(at, (1e-3, 1e-4, 1e-5, 1e-6, 1e-7)):
        size[i] = r
    x = (x * (size if tall else size[:, None])).to(dtype)
    got, ref = ops().orthogonalise(x, out_dtype=torch.float32).double(), ortho_ref(x)
    dim = 1 if tall else 2
    err = (got - ref).norm(dim=dim) / ref.norm(dim=dim)
    tol = BASE + 2.0 ** -30 * short / (41 * size.double())
    assert bool((err <= tol).all()), (err[:, at].max(0).values.tolist(), tol[at].tolist(), float(err.max()))


@pytest.mark.parametrize("shape", ORTHO)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalise_keeps_small_columns(shape, dtype):
    """columns (of the long side) 1e-3 to 1e-7 of the others"""
    x = rnd(4, *shape)
    tall = shape[1] > shape[2]
    size = torch.ones(max(shape[1:]), device="cuda")
    at = [0, 7, 17, 23, 38]
    for i, r in zip(at, (1e-3, 1e-4, 1e-5, 1e-6, 1e-7)):
        size[i] = r
    x = (x * (size[:, None] if tall else size)).to(dtype)
    got, ref = ops().orthogonalise(x, out_dtype=torch.float32).double(), ortho_ref(x)
    dim = 2 if tall else 1
    err = (got - ref).norm(dim=dim) / ref.norm(dim=dim)
    tol = BASE + 2.0 ** -40 * math.sqrt(size.numel()) / (0.3 * size.double())
    assert bool((err <= tol).all()), (err[:, at].max(0).values.tolist(), tol[at].tolist(), float(err.max()))


@pytest.mark.parametrize("shape", ORTHO)
@pytest.mark.parametrize("size,eps", [(1e-12, 1e-7), (1e-20, 1e-7), (1e-6, 1.0), (1e-9, 1e-10)])
def test_orthogonalise_of_inputs_that_eps_outweighs(shape, size, eps):
    """|x| far below eps: X0 is small, every step multiplies it by about 3.4445, and the result is as accurate as any other.
    (1e-9, 1e-10): |x| about eps"""
    x = rnd(2, *shape)
    x = x * (size / x.flatten(1).norm(dim=1).max())
    got, ref = ops().orthogonalise(x, eps=eps).double(), ortho_ref(x, eps=eps)
    err = (got - ref).flatten(1).norm(dim=1) / ref.flatten(1).norm(dim=1)
    assert float(err.max()) <= BASE, err.tolist()


@pytest.mark.parametrize("shape", [(65, 1 << 19), ((1 << 24) + 5, 1), ((1 << 20) + 1, 3), (130, (1 << 17) + 3)])
def test_orthogonalise_long_thin_matrices(shape):
    """more elements than 1024 workgroups of the usual share take"""
    x = rnd(3, *shape, dtype=torch.bfloat16).float()
    got, ref = ops().orthogonalise(x), ortho_ref(x)
    assert float((got - ref).norm() / ref.norm()) <= BASE


def muon_plain(p, g, m, v, table, lr, mu, nesterov, wd, b1, b2, eps, step):
    """the step in 64 bits, coefficients as the kernels hold them: fp32, and 1 - beta as the complement of that"""
    p, g, m, v = (t.double().clone() for t in (p, g, m, v))
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


def table_of(parts):
    rec, off = [], 0
    for q in parts:
        n = math.prod(q)
        rec.append((off, 1, 1, n, 1, 0.0, 0) if len(q) == 1 else (off,) + tuple(q) + (0, 0.2 * math.sqrt(max(q[1], q[0] * q[2])), 0))
        off += (n + 63) // 64 * 64
    return np.array(rec, dtype=ops().MUON_ENTRY), off


def muon_close(p0, p, pr, table, tol):
    """each record's update against its own size, and the roundings of p before and after"""
    for e in table:
        at = slice(int(e["off"]), int(e["off"]) + int(e["taps"]) * int(e["rows"]) * int(e["cols"]))
        a, b = p[at].double() - p0[at].double(), pr[at] - p0[at].double()
        err = float((a - b).norm())
        assert err <= tol * float(b.norm()) + 2 * U * float(pr[at].norm() + p0[at].double().norm()), (tuple(e), err, float(b.norm()))


# matrices of at least four times as many columns as rows; then with tensors longer than 1024 workgroups of the usual share
MUON = [[(1, 64, 300), (70,)], [(16, 40, 30), (5,), (9, 100, 50), (16, 130, 40), (1, 2, 9)], [(16, 512, 128), (64,)] + [(4, 300, 400)] * 9,
        [(1, 64, 300001), (20000001,)], [(4, 1, 5000001), (3,)]]


@pytest.mark.parametrize("parts", MUON)
@pytest.mark.parametrize("gbf", [False, True])
def test_muon_step_to_the_accuracy_of_its_products(parts, gbf):
    """the update of every matrix within BASE of its own size (half a step of u, in fp32, more), with fp32 and with bf16 gradients and the
    bf16 copy of the weights"""
    table, total = table_of(parts)
    p, g, m, v = rnd(10, total, scale=0.05), rnd(11, total, scale=1e-3), rnd(12, total, scale=1e-3), rnd(13, total).square() * 1e-6 + 1e-9
    if gbf:
        g = g.bfloat16()
    p0, m0, v0 = p.clone(), m.clone(), v.clone()
    pb = torch.full((total,), 7.0, dtype=torch.bfloat16, device="cuda")
    ops().muon_step(p, g, m, v, table, lr=2e-3, momentum=0.95, weight_decay=0.1, betas=(0.5, 0.999), eps=1e-8, step=4, p_bf16=pb)
    pr, mr, vr = muon_plain(p0, g, m0, v0, table, 2e-3, 0.95, True, 0.1, 0.5, 0.999, 1e-8, 4)
    muon_close(p0, p, pr, table, BASE)
    assert bool(((m.double() - mr).abs() <= 4 * U * (m0.double().abs() + g.double().abs())).all())
    assert bool(((v.double() - vr).abs() <= 8 * U * vr.abs()).all())
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for e in table:
        used[int(e["off"]):int(e["off"]) + int(e["taps"]) * int(e["rows"]) * int(e["cols"])] = True
    assert torch.equal(pb[used], p[used].bfloat16()) and bool((pb[~used] == 7).all())


# ------------------------------------------------------------------------------------------------ channel norm
@pytest.mark.parametrize("rows,ones", [(16, 16), (8192, 4)])
def test_rms_norm_backward_joins_its_sums_in_64_bits(rows, ones):
    """dgamma = 2^24 + ones - 1 from rows that lie in different groups of lanes: in fp32 every 1 would be rounded away.  The second
    form joins workgroups: two roundings to fp32"""
    h = torch.ones(rows, 200, device="cuda")
    dy = torch.zeros(rows, 200, device="cuda")
    dy[:ones] = 1.0
    dy[0] = 2.0 ** 24
    _, dgamma = ops().rms_norm_bwd(dy, h, torch.ones(rows, device="cuda"), torch.ones(200, device="cuda"))
    want = 2.0 ** 24 + ones - 1
    assert float((dgamma.double() - want).abs().max()) <= (1 if rows == 16 else 2) * U * want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("C", [96, 300, 2500])
def test_rms_norm_q8_of_rows_whose_scale_vanishes(dtype, group, C):
    """y is zero where the row's statistic is infinite: scale 1 and zero bytes, as for a group of zeros; the group with the infinity
    itself is NaN"""
    x = rnd(20, 5, C, dtype=dtype)
    x[1, 70] = float("inf")
    x[2] *= 1e30                                              # the squares pass fp32
    x[3] = 0
    q, scale, _, rstd = ops().rms_norm_q8(x, torch.ones(C, device="cuda"), group=group)
    assert float(rstd[1]) == 0 and float(rstd[2]) == 0
    back = q.float()
    for row in (2, 3):
        assert bool((scale[row] == 1).all()) and float(back[row].abs().max()) == 0
    if group == 0:
        assert bool(torch.isnan(scale[1]).all()) and bool(torch.isnan(back[1, 70]))
    else:
        k = 70 // group
        assert bool(torch.isnan(scale[1, k])) and bool(torch.isnan(back[1, 70]))
        keep = torch.arange(scale.shape[1], device="cuda") != k
        assert bool((scale[1, keep] == 1).all())
        assert float(back[1, :k * group].abs().sum()) == 0 and float(back[1, (k + 1) * group:].abs().sum()) == 0
    ok = [0, 4]
    q0, s0, _, _ = ops().rms_norm_q8(x[ok].contiguous(), torch.ones(C, device="cuda"), group=group)
    assert torch.equal(q[ok].view(torch.uint8), q0.view(torch.uint8)) and torch.equal(scale[ok], s0)


def e4m3_bytes(v):
    """round to nearest even in 64 bits (|v| <= 448): the value, and how far v is from a tie, relative to its size"""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -9))).clamp_min(-6)
    step = torch.exp2(e - 3)
    t = v / step
    return torch.round(t) * step, ((t - torch.floor(t) - 0.5).abs() * step / v.abs().clamp_min(2.0 ** -9))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C,group", [(3000, 128, 64), (500, 1030, 0), (700, 513, 32), (40, 4100, 128)])
def test_rms_norm_q8_rounds_as_the_definition_does(dtype, rows, C, group):
    """every byte against the 64-bit definition, but for values within 2^-50 of a tie of e4m3 (the rounding of fp64; rounding to fp32 first
    keeps a side of a tie or lands on it, 2^-24 more)"""
    x, r = rnd(21, rows, C, dtype=dtype), rnd(22, rows, C, dtype=dtype)
    gamma = rnd(23, C) + 1.0
    q, scale, h, _ = ops().rms_norm_q8(x, gamma, r, group=group)
    z = h.double() * gamma.double()
    g = group or C
    n = -(-C // g)
    zp = torch.nn.functional.pad(z, (0, n * g - C)).view(rows, n, g)
    v = (zp * (448.0 / zp.abs().amax(2, keepdim=True))).view(rows, n * g)[:, :C]
    want, tie = e4m3_bytes(v)
    clear = tie > 2.0 ** -23
    assert float((~clear).double().mean()) < 1e-5
    assert torch.equal(q.double()[clear], want[clear])


def test_rms_norm_q8_of_a_row_of_zeros_without_eps():
    q, scale, _, rstd = ops().rms_norm_q8(torch.zeros(2, 96, device="cuda"), torch.ones(96, device="cuda"), eps=0.0, group=32)
    assert bool(torch.isinf(rstd).all()) and bool((scale == 1).all()) and float(q.float().abs().max()) == 0


def test_rms_norm_of_rows_of_2_to_the_27_channels():
    """dgamma's join takes more columns than one launch of 1024-lane workgroups holds"""
    C = (1 << 27) + 77
    h = torch.ones(1, C, device="cuda")
    h[0, -1] = 3.0
    dy = torch.full((1, C), 2.0, device="cuda")
    one = torch.ones(1, device="cuda")
    gamma = torch.ones(C, device="cuda")
    dx, dgamma = ops().rms_norm_bwd(dy, h, one, gamma)
    assert bool((dgamma[:-1] == 2).all()) and float(dgamma[-1]) == 6
    # w - xh mean(w xh): the mean is 2 and 2^-25 more, rounded to fp32
    assert float(dx[0, :-1].abs().max()) <= 2.0 ** -22 and abs(float(dx[0, -1]) + 4) <= 2.0 ** -21
    del dx, h
    e = torch.empty(0, C, device="cuda")
    dgamma = ops().rms_norm_bwd(e, e, one[:0], gamma)[1]
    assert float(dgamma.abs().max()) == 0
    del dgamma, gamma, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", [(1, 5), (7, 64), (77, 189), (3000, 129), (300, 2048), (5, 2500), (300, 3001)])
def test_rms_norm_backward_of_a_channel_slice(dtype, rows, C):
    """x is a slice of a wider tensor and no residual is added: rms_norm hands the slice on as h, and the backward pass reads it there;
    the same numbers as from a packed copy"""
    O = ops()
    x = rnd(30, rows, C + 9, dtype=dtype)[:, 3:C + 3]
    gamma, dy, dh = rnd(31, C) + 1.0, rnd(32, rows, C, dtype=dtype), rnd(33, rows, C, dtype=dtype)
    y, h, rstd = O.rms_norm(x, gamma)
    assert h.data_ptr() == x.data_ptr()
    yc, hc, rc = O.rms_norm(x.contiguous(), gamma)
    assert torch.equal(y, yc) and torch.equal(rstd, rc)
    for d in (None, dh):
        for a, b in zip(O.rms_norm_bwd(dy, h, rstd, gamma, dh=d), O.rms_norm_bwd(dy, hc, rc, gamma, dh=d)):
            assert torch.equal(a, b)
    assert bool((y.double() - x.double() * rstd.double()[:, None] * gamma.double()).abs().max() <= 8 * float(EPS[dtype]) * float(y.abs().max()))


def test_rms_norm_module_of_a_channel_slice():
    from pose_transfer_amd.models.networks import RMSNorm
    mod = RMSNorm(40)
    wide = rnd(34, 2, 3, 5, 100)
    a, b = wide.clone().requires_grad_(), wide[..., 20:60].clone().requires_grad_()
    wy = rnd(35, 2, 3, 5, 40)
    ya, yb = mod(a[..., 20:60]), mod(b)
    assert torch.equal(ya, yb)
    ga, = torch.autograd.grad((ya * wy).sum(), a)
    gb, = torch.autograd.grad((yb * wy).sum(), b)
    assert torch.equal(ga[..., 20:60], gb) and float(ga[..., :20].abs().max()) == 0 and float(ga[..., 60:].abs().max()) == 0


# ------------------------------------------------------------------------------------------------ the trainer's recorded step
@pytest.mark.parametrize("precision", [0, 3])
@pytest.mark.parametrize("how", ["tape", "graph"])
def test_replayed_muon_step_against_the_definition(precision, how):
    """a replayed iteration's optimiser launches: each record's displacement against the 64-bit step on the arena's own gradients, at the
    step number that the device counter gives, twice; a replay that left them out, or took them twice, is off by its whole size"""
    from types import SimpleNamespace

    from pose_transfer_amd.models.pose_gan import DeformablePose_GAN
    from pose_transfer_amd.runtime import engine as E
    from pose_transfer_amd.runtime.graph import GraphedIteration
    from pose_transfer_amd.runtime.tape import TapedIteration
    from pose_transfer_amd.utils import synth
    was, E.PRECISION = E.PRECISION, precision
    try:
        opt = SimpleNamespace(image_size=(64, 64), use_input_pose=True, pose_dim=18, batch_size=2, num_stacks=4, gen_type="baseline",
                              dataset="fasion", warp_skip="mask", learning_rate=2e-4, content_loss_layer="none", nn_loss_area_size=1,
                              gan_penalty_weight=1.0, l1_penalty_weight=100.0, optimizer="muon", muon_momentum=0.9, muon_weight_decay=0.01)
        model = DeformablePose_GAN(opt, device="cuda:0")
        b = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in synth.batch(1, "muon/T", 2, 18, 64, 64)]
        b = [b[0], b[1], b[2].float().contiguous(), b[3]]
        # one eager iteration and one that is recorded and runs (tape), or two eager ones before the capture (graph)
        if how == "tape":
            replay = TapedIteration(model, [b, b, b], dict(vars(opt)), warmup=1)
        else:
            replay = GraphedIteration(model, [b, b, b], dict(vars(opt)), warmup=2)
        try:
            arenas = (model.disc.arena, model.gen.arena)
            for step in (3, 4):
                before = [(a.params.clone(), a.m.clone(), a.v.clone()) for a in arenas]
                replay.replay()
                torch.cuda.synchronize()
                for arena, (p0, m0, v0) in zip(arenas, before):
                    assert arena.step == step
                    table = arena.muon_table()
                    pr, mr, vr = muon_plain(p0, arena.grads, m0, v0, table, 2e-4, 0.9, True, 0.01, 0.5, 0.999, 1e-8, step)
                    for e in table:
                        at = slice(int(e["off"]), int(e["off"]) + int(e["taps"]) * int(e["rows"]) * int(e["cols"]))
                        a, r = arena.params[at].double() - p0[at].double(), pr[at] - p0[at].double()
                        # gradients of a real network are far from Gaussian: the products' derived bound for the matrices
                        tol = (1.5 * NS[0] ** 5 * 2.0 ** -20 if e["kind"] == 0 else 0.0) + 64 * U
                        assert float(r.norm()) > 0
                        assert float((a - r).norm()) <= tol * float(r.norm()) + 2 * U * float(pr[at].norm()) + 2 * U * float(p0[at].norm()), tuple(e)
                    assert bool(((arena.m.double() - mr).abs() <= 4 * U * (m0.double().abs() + arena.grads.double().abs())).all())
                    if precision == 3:
                        for k in arena.keys:
                            at = slice(arena.off[k], arena.off[k] + arena.numel[k])
                            assert torch.equal(arena.params_bf16[at], arena.params[at].bfloat16())
        finally:
            replay.close()
    finally:
        E.PRECISION = was
