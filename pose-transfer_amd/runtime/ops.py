"""Operators on plain tensors that do not belong to one network's schedule: the root-mean-square norm along the channels
(``rms_norm``, ``rms_norm_q8``, ``rms_norm_bwd``) and the matrix optimiser (``orthogonalise``, ``muon_step``).

Thin wrappers over the C ABI (include/posegan_hip.h): they check the arguments, allocate the outputs and the workspace
(torch's caching allocator: a captured graph gets memory of its own) and enqueue on the current stream of the tensors'
device.  No CPU fallback.  The module-level form with autograd is models/networks.py ``RMSNorm``; the trainer's optimiser
is models/pose_gan.py ``FusedMuon``."""
import ctypes as C

import numpy as np
import torch

from . import lib as L

#: include/posegan_hip.h pg_muon_entry_t: one parameter tensor of an arena (kind 0: a matrix [rows, taps * cols], 1: Adam)
MUON_ENTRY = np.dtype([("off", "<i8"), ("taps", "<i4"), ("rows", "<i4"), ("cols", "<i4"), ("kind", "<i4"), ("scale", "<f4"),
                       ("pad", "<i4")])
GROUPS = (0, 32, 64, 128, 256)
_IO = {torch.float32: 0, torch.bfloat16: 3}


class _On:
    """the tensors' device as the current one while a call enqueues (a no-op where it already is)"""

    __slots__ = ("prev", "idx")

    def __init__(self, t):
        self.prev, self.idx = None, t.get_device()

    def __enter__(self):
        cur = L.current_device()
        if cur != self.idx:
            self.prev = cur
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


# (the messages are formatted only when raised: these checks are most of a small call's host time)
def _rows(t, name, like, shape):
    """row stride of a 2-D tensor [rows, channels] of like's type and device with unit column stride"""
    if not (torch.is_tensor(t) and t.dtype == like.dtype and t.device == like.device and t.shape == shape and len(shape) == 2):
        raise ValueError("%s: %s %s on %s expected" % (name, like.dtype, tuple(shape), like.device))
    s0, s1 = t.stride()
    rows, ch = shape
    if s1 != 1 and ch > 1:
        raise ValueError("%s: channels must be contiguous" % name)
    if rows <= 1:
        return ch if ch > 0 else 1
    if s0 < ch:
        raise ValueError("%s: rows overlap" % name)
    return s0


def _vector(t, name, like, n):
    if not (torch.is_tensor(t) and t.dtype == torch.float32 and t.device == like.device and t.dim() == 1 and t.shape[0] == n
            and (n <= 1 or t.stride(0) == 1)):
        raise ValueError("%s: a contiguous fp32 vector of %d on %s expected" % (name, n, like.device))


def _channels(n):
    if n > 1 << 30:                  # the C argument has 32 bits, which ctypes would wrap
        raise ValueError("rms_norm: at most 2^30 channels")


def _norm_args(x, gamma, residual):
    if not (torch.is_tensor(x) and x.is_cuda and x.dtype in _IO and x.dim() == 2 and x.shape[1] > 0):
        raise ValueError("rms_norm: x must be an fp32 or bf16 [rows, channels] tensor on the GPU")
    shape = x.shape
    _channels(shape[1])
    _vector(gamma, "gamma", x, shape[1])
    return shape[0], shape[1], _rows(x, "x", x, shape), 0 if residual is None else _rows(residual, "residual", x, shape)


def rms_norm(x, gamma, residual=None, eps=1e-6):
    """y = h * rstd * gamma with h = x + residual (rounded to x's type), rstd = (mean_c h^2 + eps)^-1/2.
    Returns (y, h, rstd); h is x where there is no residual.  x [rows, C] fp32 or bf16, rows may be strided; gamma fp32 [C]."""
    rows, ch, ldx, ldr = _norm_args(x, gamma, residual)
    with _On(x):
        y = x.new_empty((rows, ch))
        h = None if residual is None else torch.empty_like(y)
        rstd = gamma.new_empty(rows)
        if rows:
            L.call("pg_rms_norm_fwd", x.data_ptr(), L.ptr(residual), gamma.data_ptr(), rows, ch, ldx, ldr, eps, _IO[x.dtype], L.ptr(h),
                   y.data_ptr(), ch, None, None, 0, rstd.data_ptr(), L.stream())
    return y, (x if h is None else h), rstd


def rms_norm_q8(x, gamma, residual=None, eps=1e-6, group=0):
    """the norm's output in 8 bits: (q, scale, h, rstd), q float8_e4m3fn [rows, C], value = q * scale with one fp32 scale per
    `group` channels (0: per row; scale [rows, ceil(C / group)])."""
    rows, ch, ldx, ldr = _norm_args(x, gamma, residual)
    if group not in GROUPS:
        raise ValueError("rms_norm_q8: group must be one of %s" % (GROUPS,))
    with _On(x):
        q = x.new_empty((rows, ch), dtype=torch.float8_e4m3fn)
        scale = gamma.new_empty((rows, -(-ch // group) if group else 1))
        h = None if residual is None else x.new_empty((rows, ch))
        rstd = gamma.new_empty(rows)
        if rows:
            L.call("pg_rms_norm_fwd", x.data_ptr(), L.ptr(residual), gamma.data_ptr(), rows, ch, ldx, ldr, eps, _IO[x.dtype], L.ptr(h), None,
                   0, q.data_ptr(), scale.data_ptr(), group, rstd.data_ptr(), L.stream())
    return q, scale, (x if h is None else h), rstd


def rms_norm_bwd(dy, h, rstd, gamma, dh=None):
    """(dx, dgamma) of ``rms_norm``: dx is also the residual's gradient; dh (packed): the gradient that reaches h past the norm.  h
    may be a channel slice, as ``rms_norm`` hands it on."""
    if not (torch.is_tensor(h) and h.is_cuda and h.dtype in _IO and h.dim() == 2 and h.shape[1] > 0):
        raise ValueError("rms_norm_bwd: h must be an fp32 or bf16 [rows, channels] tensor on the GPU")
    shape = h.shape
    rows, ch = shape
    _channels(ch)
    ldh = _rows(h, "h", h, shape)
    if dh is not None and _rows(dh, "dh", h, shape) != ch:
        raise ValueError("rms_norm_bwd: dh must be packed")
    lddy = _rows(dy, "dy", h, shape)
    _vector(rstd, "rstd", h, rows)
    _vector(gamma, "gamma", h, ch)
    with _On(h):
        dx = h.new_empty((rows, ch))
        dgamma = torch.empty_like(gamma)
        if rows == 0:
            return dx, dgamma.zero_()
        io = _IO[h.dtype]
        need = L.load().pg_rms_norm_bwd_workspace(rows, ch, io)
        ws = torch.empty(need, dtype=torch.uint8, device=h.device) if need else None
        L.call("pg_rms_norm_bwd_ex", dy.data_ptr(), lddy, L.ptr(dh), h.data_ptr(), ldh, rstd.data_ptr(), gamma.data_ptr(), rows, ch, io,
               dx.data_ptr(), dgamma.data_ptr(), 0, L.ptr(ws), need, L.stream())
    return dx, dgamma


def orthogonalise(x, steps=5, eps=1e-7, out_dtype=None):
    """The orthogonal factor of each matrix of x ([rows, cols] or [batch, rows, cols], fp32 or bf16) by `steps` Newton-Schulz
    products; out_dtype fp32 or bf16 (default: x's).  Accurate as fp32 products are, but for rows and columns below 1e-4 of the
    largest: a row of the short side of r is off by about 5e-11 / r of itself, a column of the long one by 1e-12 sqrt(long side) / r."""
    _need(torch.is_tensor(x) and x.is_cuda and x.dtype in _IO, "orthogonalise: x must be an fp32 or bf16 tensor on the GPU")
    _need(x.dim() in (2, 3), "orthogonalise: [rows, cols] or [batch, rows, cols] expected")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _need(out_dtype in _IO, "orthogonalise: out_dtype must be float32 or bfloat16")
    _need(1 <= steps <= 32, "orthogonalise: steps 1..32")
    x3 = x if x.dim() == 3 else x.unsqueeze(0)
    b, r, c = x3.shape
    if c > 1 and x3.stride(2) != 1 or r > 1 and x3.stride(1) < c or b > 1 and x3.stride(0) < 0:
        x3 = x3.contiguous()
    with _On(x):
        out = torch.empty((b, r, c), dtype=out_dtype, device=x.device)
        if out.numel():
            need = L.load().pg_orthogonalise_workspace(b, r, c)
            _need(need >= 0, "orthogonalise: sizes out of range")
            ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
            L.call("pg_orthogonalise", L.ptr(x3), int(x.dtype == torch.bfloat16), b, r, c, x3.stride(0) if b > 1 else 0,
                   x3.stride(1) if r > 1 else c, L.ptr(out), int(out_dtype == torch.bfloat16), r * c, c, steps, eps, L.ptr(ws), need,
                   L.stream())
    return out if x.dim() == 3 else out[0]


def muon_workspace(table):
    """bytes that a ``muon_step`` over `table` needs"""
    need = L.load().pg_muon_workspace(table.ctypes.data, len(table))
    _need(need >= 0, "muon: a tensor of the table has a size out of range")
    return need


def muon_step(p, g, m, v, table, lr, momentum=0.95, nesterov=True, weight_decay=0.0, ns_steps=5, ns_eps=1e-7, betas=(0.5, 0.999),
              eps=1e-8, step=1, grad_scale=1.0, ctr=None, p_bf16=None, workspace=None):
    """One optimiser step over a flat arena, in place on p, m (and v): the Muon update for the matrices of `table` (a numpy array
    of MUON_ENTRY records, ascending and disjoint), Adam with (betas, eps, step >= 1) for its kind 1 records.  g: fp32 or bf16 arena.
    `workspace`: a uint8 tensor of at least ``muon_workspace(table)`` bytes to use instead of a fresh one."""
    _need(isinstance(table, np.ndarray) and table.dtype == MUON_ENTRY and table.ndim == 1 and table.flags.c_contiguous,
          "muon_step: table must be a contiguous 1-D array of MUON_ENTRY records")
    _need(torch.is_tensor(p) and p.is_cuda and p.dtype == torch.float32 and p.dim() == 1 and p.is_contiguous(),
          "muon_step: p must be a contiguous fp32 arena on the GPU")
    for name, t, dts in (("g", g, (torch.float32, torch.bfloat16)), ("m", m, (torch.float32,)), ("v", v, (torch.float32,)),
                         ("p_bf16", p_bf16, (torch.bfloat16,))):
        if t is None and name in ("v", "p_bf16"):
            continue
        _need(torch.is_tensor(t) and t.dtype in dts and t.device == p.device and t.shape == p.shape and t.is_contiguous(),
              "muon_step: g, m, v and p_bf16 must be contiguous arenas like p (g fp32 or bf16, m and v fp32, p_bf16 bf16)")
    _need(1 <= ns_steps <= 32, "muon_step: ns_steps 1..32")
    _need(ctr is None or (torch.is_tensor(ctr) and ctr.dtype == torch.int64 and ctr.device == p.device and ctr.numel() >= 1),
          "muon_step: ctr must be an int64 tensor on p's device")
    if len(table) == 0:
        return
    with _On(p):
        need = muon_workspace(table)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=p.device)
        if not (workspace.dtype == torch.uint8 and workspace.device == p.device and workspace.is_contiguous() and workspace.numel() >= need):
            raise ValueError("muon_step: workspace must be a contiguous uint8 tensor of %d bytes on p's device" % need)
        d = L.MuonDesc(p=L.ptr(p), m=L.ptr(m), v=L.ptr(v), p_bf16=L.ptr(p_bf16), entries=table.ctypes.data, total=p.numel(),
                       n=len(table), nesterov=int(bool(nesterov)), steps=ns_steps, lr=lr, momentum=momentum, weight_decay=weight_decay,
                       grad_scale=grad_scale, eps=ns_eps, beta1=betas[0], beta2=betas[1], adam_eps=eps, step=step, ctr=L.ptr(ctr),
                       workspace=L.ptr(workspace), workspace_bytes=workspace.numel())
        if g.dtype == torch.bfloat16:
            d.g_bf16 = L.ptr(g)
        else:
            d.g = L.ptr(g)
        L.call("pg_muon_step", C.byref(d), L.stream())
