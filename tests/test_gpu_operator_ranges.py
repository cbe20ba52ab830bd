"""Range and edge tests of the channel norm and the matrix optimiser (runtime/ops.py) beside tests/test_gpu_operators.py, against plain
implementations in 64 bits.

Tolerances.  U = 2^-24, EPS the half step of the stored type.
  orthogonal factor, inputs whose long side is at least four times the short one: a Gaussian's singular values then lie within a factor
      (1 + 1/2) / (1 - 1/2) = 3 of each other.  A step has four products of 22-bit operands, each within 2^-21 of its size; twenty of them,
      magnified by at most that factor: BASE = 20 * 2^-21 * 3 = 2.9e-5.  (Operands of 11 bits, one of the two fp16 values lost, are
      ten times outside.)
  rows much smaller than the others: the m x m factor P of a stage is off by an absolute 2^-30 at most (G by 2^-40, Q by 4.8 times that
      and 2^-39 of its own, three of them multiplied: 36 times, then P's own 2^-35 twice), so a row by 2^-30 sqrt(m) |X|_2, |X|_2 <= 1; the
      row itself, r of the others, grows from r / sqrt(m) to 41 times that: relative 2^-30 m / (41 r)."""
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
@pytest.mark.parametrize("size,eps", [(1e-12, 1e-7), (1e-20, 1e-7), (1e-6, 1.0), (1e-9, 1e-10)])
def test_orthogonalise_of_inputs_that_eps_outweighs(shape, size, eps):
    """|x| far below eps: X0 is small, every step multiplies it by about 3.4445, and the result is as accurate as any other.
    (1e-9, 1e-10): |x| about eps"""
    x = rnd(2, *shape)
    x = x * (size / x.flatten(1).norm(dim=1).max())
    got, ref = ops().orthogonalise(x, eps=eps).double(), ortho_ref(x, eps=eps)
    err = (got - ref).flatten(1).norm(dim=1) / ref.flatten(1).norm(dim=1)
    assert float(err.max()) <= BASE, err.tolist()
