"""The cases on which the channel norm (root mean square, with the residual's addition) and the matrix optimiser
(Newton-Schulz orthogonalisation, Muon step) are measured.

``run`` computes an operator in plain 32-bit torch where ``own`` is false and through the framework's entry points
(pose-transfer_amd/runtime/ops.py over include/posegan_hip.h) where it is true.  ``exact`` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

NS = (3.4445, -4.7750, 2.0315)          # the quintic a s + b s^3 + c s^5 of the orthogonalisation
NS_STEPS, NS_EPS = 5, 1e-7
RMS_EPS = 1e-6
MU, LR, WD = 0.95, 2e-3, 0.01           # Muon: momentum, learning rate, decoupled decay
B1, B2, ADAM_EPS = 0.5, 0.999, 1e-8     # the trainer's Adam, for the tensors that are no matrices
E4M3_MAX = 448.0

#: one record per parameter tensor of an arena: kind 0 = a matrix [rows, taps * cols] stored [taps][rows][cols], kind 1 = a vector (Adam)
ENTRY = np.dtype([("off", "<i8"), ("taps", "<i4"), ("rows", "<i4"), ("cols", "<i4"), ("kind", "<i4"), ("scale", "<f4"), ("pad", "<i4")])

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}

# the generator's and the discriminator's inner convolutions at 256 x 256: taps x Cout x Cin each (two encoders; the decoder
# reads three concatenated sources), and the vectors between them
_ENC = "16x128x64,16x256x128,16x512x256,16x512x512,16x512x512,16x512x512"
_GEN256 = ",".join([_ENC, _ENC, "16x512x1024,16x512x1536,16x512x1536,16x512x1536,16x256x1024,16x128x512", "v11520,v7000,v6912,v64"])
_DISC256 = "16x128x64,16x256x128,16x512x256,v43008,v8192,v64"


def listed():
    return [
        # one pixel's channels: what a serving loop or a 1 x 1 bottleneck map hands over; launch latency
        {"name": "rms_fwd_row", "op": "rms_fwd", "rows": 1, "C": 512, "dtype": "bf16", "res": True, "group": 0, "ld": 512},
        # batch 4 at 64 x 64 x 256 in fp32 storage
        {"name": "rms_fwd_f32", "op": "rms_fwd", "rows": 16384, "C": 256, "dtype": "f32", "res": True, "group": -1, "ld": 256},
        # the decoder's concatenation at 64 x 64, batch 32: x is a channel slice of a wider tensor, no residual
        {"name": "rms_fwd_slice", "op": "rms_fwd", "rows": 131072, "C": 513, "dtype": "bf16", "res": False, "group": -1, "ld": 1026},
        # batch 32 at 128 x 128 x 128 in bf16, kept in 8 bits with a scale per 64 channels
        {"name": "rms_fwd_q8", "op": "rms_fwd", "rows": 524288, "C": 128, "dtype": "bf16", "res": True, "group": 64, "ld": 128},
        # a small ragged backward in fp32
        {"name": "rms_bwd_small", "op": "rms_bwd", "rows": 77, "C": 189, "dtype": "f32", "res": True},
        # batch 32 at 64 x 64 x 512 in bf16 storage
        {"name": "rms_bwd_bf16", "op": "rms_bwd", "rows": 131072, "C": 512, "dtype": "bf16", "res": True},
        # one small layer: latency of the chain of products
        {"name": "orth_small", "op": "orth", "batch": 1, "rows": 64, "cols": 162, "dtype": "bf16"},
        # the taps of one odd-sized tall layer, each as its own matrix
        {"name": "orth_tall", "op": "orth", "batch": 16, "rows": 770, "cols": 189, "dtype": "f32"},
        # the widest decoder layer, flattened
        {"name": "orth_wide", "op": "orth", "batch": 1, "rows": 512, "cols": 24576, "dtype": "bf16"},
        # the optimiser step of the discriminator and of the generator at 256 x 256
        {"name": "muon_disc", "op": "muon", "tensors": _DISC256, "nesterov": True},
        {"name": "muon_gen", "op": "muon", "tensors": _GEN256, "nesterov": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms_fwd", "rms_bwd", "orth", "muon"])
    if op in ("rms_fwd", "rms_bwd"):
        C = _log_int(rng, 8, 1536)
        rows = _log_int(rng, 1, max(1, (60 << 20) // C))
        case = {"op": op, "rows": rows, "C": C, "dtype": rng.choice(["f32", "bf16"]), "res": rng.random() < 0.6}
        if op == "rms_fwd":
            case["group"] = rng.choice([-1, -1, 0, 32, 64, 128])
            case["ld"] = C + rng.choice([0, 0, 8, 24, C])
        return case
    if op == "orth":
        rows, cols = _log_int(rng, 1, 1024), _log_int(rng, 1, 8192)
        if rng.random() < 0.3:
            rows, cols = cols, rows
        cost = min(rows, cols) ** 2 * max(rows, cols)
        return {"op": op, "batch": _log_int(rng, 1, max(1, min(64, (6 << 30) // max(1, cost)))), "rows": rows, "cols": cols,
                "dtype": rng.choice(["f32", "bf16"])}
    parts = []
    for _ in range(rng.randint(1, 8)):
        if rng.random() < 0.25:
            parts.append("v%d" % _log_int(rng, 1, 50000))
        else:
            parts.append("%dx%dx%d" % (rng.choice([1, 9, 16]), _log_int(rng, 2, 512), _log_int(rng, 2, 1024)))
    return {"op": op, "tensors": ",".join(parts), "nesterov": rng.random() < 0.7}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 11)
    return g


def _table(tensors):
    """the arena's records; every tensor starts at a multiple of 64 elements, as in the trainer's arenas"""
    rec, off = [], 0
    for t in tensors.split(","):
        if t[0] == "v":
            n, r = int(t[1:]), (off, 1, 1, int(t[1:]), 1, 0.0, 0)
        else:
            taps, rows, cols = (int(v) for v in t.split("x"))
            n = taps * rows * cols
            # update of root mean square 0.2: the same learning rate serves the Adam tensors
            r = (off, taps, rows, cols, 0, 0.2 * math.sqrt(max(rows, taps * cols)), 0)
        rec.append(r)
        off += (n + 63) // 64 * 64
    return np.array(rec, dtype=ENTRY), off


def _gradient(g, rows, cols, batch=1):
    """gradients of a layer: a few strong directions over a noise floor, and channels of uneven size"""
    k = max(1, min(rows, cols) // 8)
    u = torch.randn(batch, rows, k, device="cuda", generator=g)
    v = torch.randn(batch, k, cols, device="cuda", generator=g)
    x = torch.randn(batch, rows, cols, device="cuda", generator=g) + torch.matmul(u, v).mul_(1.0 / math.sqrt(k))
    return x * (0.5 + torch.rand(batch, rows, 1, device="cuda", generator=g)) * 1e-3


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op in ("rms_fwd", "rms_bwd"):
        rows, C, dt = case["rows"], case["C"], DTYPE[case["dtype"]]
        s = {"case": case, "gamma": 1.0 + 0.2 * torch.randn(C, device="cuda", generator=g)}
        size = torch.exp2(torch.randn(rows, 1, device="cuda", generator=g))        # pixels of uneven size
        if op == "rms_fwd":
            ld = case["ld"]
            s["x"] = (torch.randn(rows, ld, device="cuda", generator=g) * size).to(dt)[:, :C]
            s["res"] = torch.randn(rows, C, device="cuda", generator=g).to(dt) if case["res"] else None
            return s
        h = (torch.randn(rows, C, device="cuda", generator=g) * size).to(dt)
        s["h"] = h
        s["rstd"] = torch.rsqrt(h.double().square().mean(1) + RMS_EPS).float()         # saved by the forward pass
        s["dy"] = torch.randn(rows, C, device="cuda", generator=g).to(dt)
        s["dh"] = torch.randn(rows, C, device="cuda", generator=g).to(dt) if case["res"] else None
        return s
    if op == "orth":
        return {"case": case, "x": _gradient(g, case["rows"], case["cols"], case["batch"]).to(DTYPE[case["dtype"]])}
    table, total = _table(case["tensors"])
    s = {"case": case, "table": table, "t": 3, "total": total}
    for k in ("p", "g", "m", "v"):
        s[k] = torch.zeros(total, device="cuda")
    for e in table:
        n = int(e["taps"]) * int(e["rows"]) * int(e["cols"])
        at = slice(int(e["off"]), int(e["off"]) + n)
        if e["kind"] == 0:
            flat = int(e["taps"]) * int(e["cols"])
            bound = math.sqrt(6.0 / (flat + int(e["rows"]) * int(e["taps"])))          # Glorot, as the trainer starts
            s["p"][at] = (torch.rand(n, device="cuda", generator=g) * 2 - 1) * bound
            for k in ("g", "m"):
                x = _gradient(g, int(e["rows"]), flat)[0]
                s[k][at] = x.view(int(e["rows"]), int(e["taps"]), int(e["cols"])).permute(1, 0, 2).reshape(-1)
        else:
            s["p"][at] = torch.randn(n, device="cuda", generator=g) * 0.05
            s["g"][at] = torch.randn(n, device="cuda", generator=g) * 1e-3
            s["m"][at] = torch.randn(n, device="cuda", generator=g) * 1e-3
            s["v"][at] = torch.rand(n, device="cuda", generator=g) * 1e-6 + 1e-8
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _rms_fwd(s):
    c = s["case"]
    h = s["x"].float()
    if s["res"] is not None:
        h = h + s["res"].float()
    h = h.to(s["x"].dtype)                                  # the stored sum is what the norm and its backward read
    f = h.float()
    rstd = torch.rsqrt(f.square().mean(1) + RMS_EPS)
    y = f * rstd[:, None] * s["gamma"]
    out = {"rstd": rstd}
    if c["res"]:
        out["h"] = h
    if c["group"] < 0:
        out["y"] = y.to(h.dtype)
        return out
    rows, C = y.shape
    grp = c["group"] or C
    n = -(-C // grp)
    yp = torch.nn.functional.pad(y, (0, n * grp - C)).view(rows, n, grp)
    amax = yp.abs().amax(2)
    scale = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    q = (yp / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows, n * grp)[:, :C]
    out["q"], out["scale"] = q.to(torch.float8_e4m3fn).contiguous(), scale
    return out


def _rms_bwd(s):
    f, dy = s["h"].float(), s["dy"].float()
    xh = f * s["rstd"][:, None]
    w = dy * s["gamma"]
    dx = (w - xh * (w * xh).mean(1, keepdim=True)) * s["rstd"][:, None]
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    # long sums of either sign: in 64 bits
    return {"dx": dx.to(s["h"].dtype), "dgamma": (dy * xh).sum(0, dtype=torch.float64).float()}


def _newton_schulz(x):
    """x: [batch, rows, cols] in 32 bits"""
    wide = x if x.shape[1] <= x.shape[2] else x.transpose(1, 2).contiguous()
    wide = wide / (wide.square().sum((1, 2), keepdim=True, dtype=torch.float64).sqrt().float() + NS_EPS)
    a, b, c = NS
    for _ in range(NS_STEPS):                               # each step needs the one before
        A = torch.matmul(wide, wide.transpose(1, 2).contiguous())
        wide = a * wide + torch.matmul(b * A + c * torch.matmul(A, A), wide)
    return wide if x.shape[1] <= x.shape[2] else wide.transpose(1, 2)


def _muon(s):
    p, g, m, v = s["p"], s["g"], s["m"], s["v"]
    for e in s["table"]:                                    # tensors of different shapes
        taps, rows, cols = int(e["taps"]), int(e["rows"]), int(e["cols"])
        at = slice(int(e["off"]), int(e["off"]) + taps * rows * cols)
        if e["kind"] == 0:
            m[at] = MU * m[at] + (1 - MU) * g[at]
            u = (1 - MU) * g[at] + MU * m[at] if s["case"]["nesterov"] else m[at]
            x = u.view(taps, rows, cols).permute(1, 0, 2).reshape(1, rows, taps * cols)
            o = _newton_schulz(x)[0].reshape(rows, taps, cols).permute(1, 0, 2).reshape(-1)
            p[at] = p[at] * (1 - LR * WD) - LR * float(e["scale"]) * o
        else:
            m[at] = B1 * m[at] + (1 - B1) * g[at]
            v[at] = B2 * v[at] + (1 - B2) * g[at] * g[at]
            den = v[at].sqrt() / math.sqrt(1 - B2 ** s["t"]) + ADAM_EPS
            p[at] = p[at] - LR / (1 - B1 ** s["t"]) * m[at] / den
    return {"p": p, "m": m, "v": v}


def run(state):
    c = state["case"]
    if not own:
        if c["op"] == "orth":
            return {"o": _newton_schulz(state["x"].float()).to(torch.bfloat16).contiguous()}
        return {"rms_fwd": _rms_fwd, "rms_bwd": _rms_bwd, "muon": _muon}[c["op"]](state)
    ops = _ops()
    if c["op"] == "rms_fwd":
        if c["group"] < 0:
            y, h, rstd = ops.rms_norm(state["x"], state["gamma"], state["res"], eps=RMS_EPS)
            out = {"rstd": rstd, "y": y}
        else:
            q, scale, h, rstd = ops.rms_norm_q8(state["x"], state["gamma"], state["res"], eps=RMS_EPS, group=c["group"])
            out = {"rstd": rstd, "q": q, "scale": scale}
        if c["res"]:
            out["h"] = h
        return out
    if c["op"] == "rms_bwd":
        dx, dgamma = ops.rms_norm_bwd(state["dy"], state["h"], state["rstd"], state["gamma"], dh=state["dh"])
        return {"dx": dx, "dgamma": dgamma}
    if c["op"] == "orth":
        return {"o": ops.orthogonalise(state["x"], steps=NS_STEPS, eps=NS_EPS, out_dtype=torch.bfloat16)}
    ops.muon_step(state["p"], state["g"], state["m"], state["v"], state["table"], lr=LR, momentum=MU, nesterov=c["nesterov"],
                  weight_decay=WD, ns_steps=NS_STEPS, ns_eps=NS_EPS, betas=(B1, B2), eps=ADAM_EPS, step=state["t"])
    return {"p": state["p"], "m": state["m"], "v": state["v"]}


_loaded = []


def _ops():
    if not _loaded:
        import pta_bootstrap
        pta_bootstrap.load()
        from pose_transfer_amd.runtime import ops
        _loaded.append(ops)
    return _loaded[0]


# ------------------------------------------------------------------------------------------------ cost and definition
def work(case):
    op = case["op"]
    if op in ("rms_fwd", "rms_bwd"):
        n, b = case["rows"] * case["C"], 4 if case["dtype"] == "f32" else 2
        if op == "rms_bwd":
            return {"bytes": n * b * (4 if case["res"] else 3) + 4 * case["rows"] + 8 * case["C"], "flops": 12 * n}
        out = n * b if case["group"] < 0 else n + 4 * case["rows"] * -(-case["C"] // (case["group"] or case["C"]))
        return {"bytes": n * b * (3 if case["res"] else 1) + out + 4 * case["rows"] + 4 * case["C"], "flops": 6 * n}
    if op == "orth":
        m, n = sorted((case["rows"], case["cols"]))
        return {"bytes": case["batch"] * m * n * (2 + (4 if case["dtype"] == "f32" else 2)), "flops": case["batch"] * _ns_flops(m, n)}
    table, _ = _table(case["tensors"])
    total = {"bytes": 0, "flops": 0}
    for e in table:
        n = int(e["taps"]) * int(e["rows"]) * int(e["cols"])
        total["bytes"] += n * (20 if e["kind"] == 0 else 28)
        total["flops"] += 8 * n
        if e["kind"] == 0:
            total["flops"] += _ns_flops(*sorted((int(e["rows"]), int(e["taps"]) * int(e["cols"]))))
    return total


def _ns_flops(m, n):
    """least: the Gram matrix (half of it), the polynomial in it (four symmetric products a step), one product with the matrix"""
    return m * m * n + 4 * NS_STEPS * m ** 3 + 2 * m * m * n


def _orthogonal64(x):
    """x: one matrix in 64 bits.  Every iterate is a polynomial of x x^T times x: Horner's form on the short side"""
    tall = x.shape[0] > x.shape[1]
    z = (x.t() if tall else x) / (torch.linalg.vector_norm(x) + NS_EPS)
    a, b, c = NS
    eye = torch.eye(z.shape[0], dtype=torch.float64, device=z.device)
    for _ in range(NS_STEPS):
        A = z @ z.t().contiguous()
        z = (a * eye + A @ (b * eye + c * A)) @ z
    return z.t() if tall else z


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "orth":
        return {"o": torch.stack([_orthogonal64(x) for x in s["x"].double()])}
    if op == "muon":
        out = {k: s[k].double() for k in ("p", "m", "v")}
        for e in s["table"]:
            taps, rows, cols = int(e["taps"]), int(e["rows"]), int(e["cols"])
            at = slice(int(e["off"]), int(e["off"]) + taps * rows * cols)
            g = s["g"][at].double()
            if e["kind"] == 1:
                out["m"][at] = out["m"][at] + (1 - B1) * (g - out["m"][at])
                out["v"][at] = out["v"][at] + (1 - B2) * (g * g - out["v"][at])
                step = (out["m"][at] / (1 - B1 ** s["t"])) / ((out["v"][at] / (1 - B2 ** s["t"])).sqrt() + ADAM_EPS)
                out["p"][at] -= LR * step
                continue
            out["m"][at] = out["m"][at] + (1 - MU) * (g - out["m"][at])
            u = g + MU * (out["m"][at] - g) if case["nesterov"] else out["m"][at]
            x = torch.cat(list(u.view(taps, rows, cols)), dim=1)
            o = torch.stack(list(_orthogonal64(x).split(cols, dim=1)))
            out["p"][at] -= LR * (WD * out["p"][at] + float(e["scale"]) * o.reshape(-1))
        return out
    gamma = s["gamma"].double()
    if op == "rms_bwd":
        h, dy = s["h"].double(), s["dy"].double()
        C = h.shape[1]
        r = s["rstd"].double()[:, None]
        dot = (dy * gamma * h).sum(1, keepdim=True)
        dx = r * dy * gamma - r ** 3 * h * dot / C
        if s["dh"] is not None:
            dx = dx + s["dh"].double()
        return {"dx": dx, "dgamma": torch.einsum("rc,rc->c", dy, h * r)}
    h = s["x"].double() if s["res"] is None else s["x"].double() + s["res"].double()
    if s["x"].dtype == torch.bfloat16:
        h = h.float().to(torch.bfloat16).double()            # sums of two bf16 values are exact in 32 bits but for the last places
    r = 1.0 / torch.sqrt(torch.einsum("rc,rc->r", h, h) / h.shape[1] + RMS_EPS)
    y = h * gamma * r[:, None]
    out = {"rstd": r}
    if case["res"]:
        out["h"] = h
    if case["group"] < 0:
        out["y"] = y
        return out
    grp = case["group"] or y.shape[1]
    scales, qs = [], []
    for part in y.split(grp, dim=1):
        top = part.abs().max(dim=1, keepdim=True).values
        sc = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        scales.append(sc)
        qs.append((part / sc).float().to(torch.float8_e4m3fn).double())
    out["q"], out["scale"] = torch.cat(qs, 1), torch.cat(scales, 1)
    return out
