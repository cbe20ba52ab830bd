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

    def __init__(self, device):
        self.prev, self.idx = None, device.index

    def __enter__(self):
        cur = torch.cuda.current_device()
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


def _rows(t, name, dtype, device, shape=None):
    """a 2-D tensor with unit column stride; its row stride"""
    _need(torch.is_tensor(t) and t.dim() == 2, "%s: a 2-D tensor [rows, channels] is required" % name)
    _need(t.dtype == dtype and t.device == device, "%s: %s on %s expected, got %s on %s" % (name, dtype, device, t.dtype, t.device))
    _need(shape is None or tuple(t.shape) == tuple(shape), "%s: shape %s expected, got %s" % (name, shape and tuple(shape), tuple(t.shape)))
    _need(t.shape[1] <= 1 or t.stride(1) == 1, "%s: channels must be contiguous" % name)
    ld = t.stride(0) if t.shape[0] > 1 else max(1, t.shape[1])
    _need(ld >= t.shape[1], "%s: rows overlap" % name)
    return ld


def _norm_args(x, gamma, residual):
    _need(torch.is_tensor(x) and x.is_cuda and x.dtype in _IO, "rms_norm: x must be an fp32 or bf16 tensor on the GPU")
    ldx = _rows(x, "x", x.dtype, x.device)
    rows, ch = x.shape
    _need(ch > 0, "rms_norm: no channels")
    _need(torch.is_tensor(gamma) and gamma.dtype == torch.float32 and gamma.device == x.device and tuple(gamma.shape) == (ch,)
          and (ch == 1 or gamma.stride(0) == 1), "rms_norm: gamma must be a contiguous fp32 [%d] on x's device" % ch)
    ldr = 0 if residual is None else _rows(residual, "residual", x.dtype, x.device, x.shape)
    return rows, ch, ldx, ldr


def rms_norm(x, gamma, residual=None, eps=1e-6):
    """y = h * rstd * gamma with h = x + residual (rounded to x's type), rstd = (mean_c h^2 + eps)^-1/2.
    Returns (y, h, rstd); h is x where there is no residual.  x [rows, C] fp32 or bf16, rows may be strided; gamma fp32 [C]."""
    rows, ch, ldx, ldr = _norm_args(x, gamma, residual)
    with _On(x.device):
        y = torch.empty((rows, ch), dtype=x.dtype, device=x.device)
        h = torch.empty_like(y) if residual is not None else None
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        if rows:
            L.call("pg_rms_norm_fwd", L.ptr(x), L.ptr(residual), L.ptr(gamma), rows, ch, ldx, ldr, eps, _IO[x.dtype], L.ptr(h),
                   L.ptr(y), ch, None, None, 0, L.ptr(rstd), L.stream())
    return y, (x if h is None else h), rstd


def rms_norm_q8(x, gamma, residual=None, eps=1e-6, group=0):
    """the norm's output in 8 bits: (q, scale, h, rstd), q float8_e4m3fn [rows, C], value = q * scale with one fp32 scale per
    `group` channels (0: per row; scale [rows, ceil(C / group)])."""
    rows, ch, ldx, ldr = _norm_args(x, gamma, residual)
    _need(group in GROUPS, "rms_norm_q8: group must be one of %s" % (GROUPS,))
    with _On(x.device):
        q = torch.empty((rows, ch), dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty((rows, -(-ch // group) if group else 1), dtype=torch.float32, device=x.device)
        h = torch.empty((rows, ch), dtype=x.dtype, device=x.device) if residual is not None else None
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        if rows:
            L.call("pg_rms_norm_fwd", L.ptr(x), L.ptr(residual), L.ptr(gamma), rows, ch, ldx, ldr, eps, _IO[x.dtype], L.ptr(h), None,
                   0, L.ptr(q), L.ptr(scale), group, L.ptr(rstd), L.stream())
    return q, scale, (x if h is None else h), rstd


def rms_norm_bwd(dy, h, rstd, gamma, dh=None):
    """(dx, dgamma) of ``rms_norm``: dx is also the residual's gradient; dh: the gradient that reaches h past the norm."""
    _need(torch.is_tensor(h) and h.is_cuda and h.dtype in _IO, "rms_norm_bwd: h must be an fp32 or bf16 tensor on the GPU")
    rows, ch = h.shape if h.dim() == 2 else (0, 0)
    _need(ch > 0 and _rows(h, "h", h.dtype, h.device) == ch, "rms_norm_bwd: h must be a packed [rows, C] tensor")
    lddy = _rows(dy, "dy", h.dtype, h.device, h.shape)
    _need(dh is None or _rows(dh, "dh", h.dtype, h.device, h.shape) == ch, "rms_norm_bwd: dh must be packed")
    for name, t, n in (("rstd", rstd, rows), ("gamma", gamma, ch)):
        _need(torch.is_tensor(t) and t.dtype == torch.float32 and t.device == h.device and tuple(t.shape) == (n,)
              and (n <= 1 or t.stride(0) == 1), "rms_norm_bwd: %s must be a contiguous fp32 [%d] on h's device" % (name, n))
    with _On(h.device):
        dx = torch.empty((rows, ch), dtype=h.dtype, device=h.device)
        dgamma = torch.empty(ch, dtype=torch.float32, device=h.device)
        if rows == 0:
            return dx, dgamma.zero_()
        need = L.load().pg_rms_norm_bwd_workspace(rows, ch, _IO[h.dtype])
        ws = torch.empty(need, dtype=torch.uint8, device=h.device) if need else None
        L.call("pg_rms_norm_bwd", L.ptr(dy), lddy, L.ptr(dh), L.ptr(h), L.ptr(rstd), L.ptr(gamma), rows, ch, _IO[h.dtype], L.ptr(dx),
               L.ptr(dgamma), 0, L.ptr(ws), need, L.stream())
    return dx, dgamma


def orthogonalise(x, steps=5, eps=1e-7, out_dtype=None):
    """The orthogonal factor of each matrix of x ([rows, cols] or [batch, rows, cols], fp32 or bf16) by `steps` Newton-Schulz
    products; fp32 accuracy inside, out_dtype fp32 or bf16 (default: x's)."""
    _need(torch.is_tensor(x) and x.is_cuda and x.dtype in _IO, "orthogonalise: x must be an fp32 or bf16 tensor on the GPU")
    _need(x.dim() in (2, 3), "orthogonalise: [rows, cols] or [batch, rows, cols] expected")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _need(out_dtype in _IO, "orthogonalise: out_dtype must be float32 or bfloat16")
    x3 = x if x.dim() == 3 else x.unsqueeze(0)
    b, r, c = x3.shape
    if c > 1 and x3.stride(2) != 1 or r > 1 and x3.stride(1) < c or b > 1 and x3.stride(0) < 0:
        x3 = x3.contiguous()
    with _On(x.device):
        out = torch.empty((b, r, c), dtype=out_dtype, device=x.device)
        if out.numel():
            need = L.load().pg_orthogonalise_workspace(b, r, c)
            _need(need >= 0, "orthogonalise: sizes out of range")
            ws = torch.empty(need, dtype=torch.uint8, device=x.device)
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
    of MUON_ENTRY records, ascending and disjoint), Adam with (betas, eps, step) for its kind 1 records.  g: fp32 or bf16 arena.
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
              "muon_step: %s must be a contiguous arena like p" % name)
    _need(ctr is None or (torch.is_tensor(ctr) and ctr.dtype == torch.int64 and ctr.device == p.device and ctr.numel() >= 1),
          "muon_step: ctr must be an int64 tensor on p's device")
    if len(table) == 0:
        return
    with _On(p.device):
        need = muon_workspace(table)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=p.device)
        _need(workspace.dtype == torch.uint8 and workspace.device == p.device and workspace.is_contiguous() and workspace.numel() >= need,
              "muon_step: workspace must be a contiguous uint8 tensor of %d bytes on p's device" % need)
        d = L.MuonDesc(p=L.ptr(p), m=L.ptr(m), v=L.ptr(v), p_bf16=L.ptr(p_bf16), entries=table.ctypes.data, total=p.numel(),
                       n=len(table), nesterov=int(bool(nesterov)), steps=ns_steps, lr=lr, momentum=momentum, weight_decay=weight_decay,
                       grad_scale=grad_scale, eps=ns_eps, beta1=betas[0], beta2=betas[1], adam_eps=eps, step=step, ctr=L.ptr(ctr),
                       workspace=L.ptr(workspace), workspace_bytes=workspace.numel())
        if g.dtype == torch.bfloat16:
            d.g_bf16 = L.ptr(g)
        else:
            d.g = L.ptr(g)
        L.call("pg_muon_step", C.byref(d), L.stream())
