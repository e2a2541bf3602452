"""64-bit forms of the dense operators, with bounds on how far a result in fewer bits may be.

Every function works on CPU float64 tensors.  The bounds follow the arithmetic of the kernels:
u is the relative error of one rounding to the storage type (bf16 2^-8, fp32 2^-24) and a
product summed over n terms in fp32 is off by at most (n + 2) 2^-23 of the sum of the absolute
terms (an addition on the tensor cores may truncate, hence 2^-23 and not 2^-24).  The fast
exponential, logarithm and division of the bf16 path are within 2^-18 of the activation's
scale; fp32 uses the accurate ones, within 2^-21.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SUM = 2.0 ** -23
# 1.2 bounds |act'| and |z act''(z)| of every activation here at gamma 0.1 (gelu' <= 1.13,
# softplus' <= 1, |z gelu''| <= 1.1)
SLOPE, CURVE = 1.25, 1.25


def act(z, kind, gamma):
    if kind == "none":
        return z
    if kind == "relu":
        return torch.clamp(z, min=0)
    if kind == "silu":
        return z * torch.sigmoid(z)
    g = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if kind == "gelu_tanh":
        return g
    return g + gamma * torch.where(z > 20, z, torch.log1p(torch.exp(torch.clamp(z, max=20))))


def act_grad(z, kind, gamma):
    if kind == "none":
        return torch.ones_like(z)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    c, a = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(c * (z + a * z ** 3))
    d = 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * a * z * z)
    if kind == "gelu_tanh":
        return d
    return d + gamma * torch.where(z > 20, torch.ones_like(z), torch.sigmoid(z))


def approx(dtype):
    return 2.0 ** -18 if dtype == torch.bfloat16 else 2.0 ** -21


def product(a, b, ea=None, eb=None):
    """(a @ b, its bound): operands off by ea and eb, the sum accumulated in fp32."""
    n = a.shape[-1]
    bound = (n + 2) * SUM * (a.abs() @ b.abs())
    if ea is not None:
        bound = bound + ea @ b.abs()
    if eb is not None:
        bound = bound + a.abs() @ eb
    if ea is not None and eb is not None:
        bound = bound + ea @ eb
    return a @ b, bound


def affine(x, w, b):
    z, e = product(x, w.t())
    if b is not None:
        z = z + b
        e = e + SUM * z.abs()
    return z, e


def linear(x, w, b, r, dy, kind, gamma, dtype, grad_dtype=None):
    """{name: (value, bound)} of y, dx, dw, db."""
    u, up = U[dtype], U[grad_dtype or dtype]
    f = approx(dtype)
    z, ez = affine(x, w, b)
    a = act(z, kind, gamma)
    ea = SLOPE * ez + (0 if kind == "none" else f * (z.abs() + 1))
    y = a if r is None else a + r
    ey = ea + SUM * y.abs()
    out = {"y": (y, ey + u * (y.abs() + ey))}
    if dy is None:
        return out
    d = act_grad(z, kind, gamma)
    dz = dy * d
    if kind == "none":
        edz = torch.zeros_like(dz)
    else:  # z is kept rounded, dz is stored rounded
        ed = CURVE * (u + ez / z.abs().clamp(min=1e-30)).clamp(max=1.0) + 8 * f
        if kind == "relu":  # the sign of z is only in doubt within its error
            ed = (z.abs() <= ez).to(z.dtype)
        edz = dy.abs() * ed
        edz = edz + u * (dz.abs() + edz)
    n = dz.shape[0]
    dx, edx = product(dz, w, edz)
    dw, edw = product(dz.t(), x, edz.t())
    # the bias gradient sums unrounded dz in fp32
    db, edb = dz.sum(0), edz.sum(0) + (n + 2) * SUM * dz.abs().sum(0)
    out["dx"] = (dx, edx + u * (dx.abs() + edx))
    out["dw"] = (dw, edw + up * (dw.abs() + edw))
    out["db"] = (db, edb + up * (db.abs() + edb))
    return out


def gated_ffn(x, wg, wu, wd, bg, bu, bd, r, dy, kind, gamma, dtype, grad_dtype=None):
    """{name: (value, bound)} of y, dx, dwg, dwu, dwd, dbg, dbu, dbd."""
    u, up = U[dtype], U[grad_dtype or dtype]
    f = approx(dtype)
    g, eg = affine(x, wg, bg)
    v, ev = affine(x, wu, bu)
    a = act(g, kind, gamma)
    ea = SLOPE * eg + f * (g.abs() + 1)
    h = a * v
    eh = ea * v.abs() + a.abs() * ev + ea * ev + SUM * h.abs()
    eh = eh + u * (h.abs() + eh)  # h is stored rounded
    y, ey = product(h, wd.t(), eh)
    for t in (bd, r):
        if t is not None:
            y = y + t
            ey = ey + SUM * y.abs()
    out = {"y": (y, ey + u * (y.abs() + ey))}
    if dy is None:
        return out
    dh, edh = product(dy, wd)
    # g and u (v here) are kept in fp32
    d = act_grad(g, kind, gamma)
    ed = CURVE * (eg / g.abs().clamp(min=1e-30)).clamp(max=1.0) + 8 * f
    if kind == "relu":
        ed = (g.abs() <= eg).to(g.dtype)
    ea = SLOPE * eg + f * (g.abs() + 1)

    def times(p, ep, q, eq):
        return p * q, ep * q.abs() + p.abs() * eq + ep * eq + SUM * (p * q).abs()

    du, edu = times(dh, edh, a, ea)
    dg, edg = times(*times(dh, edh, v, ev), d, ed)
    edu, edg = edu + u * (du.abs() + edu), edg + u * (dg.abs() + edg)
    p1, e1 = product(dg, wg, edg)
    p2, e2 = product(du, wu, edu)
    n = 2 * wg.shape[0]
    dx, edx = p1 + p2, e1 + e2 + n * SUM * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    out["dx"] = (dx, edx + u * (dx.abs() + edx))
    for name, (p, ep, q, eq) in {"dwg": (dg, edg, x, None), "dwu": (du, edu, x, None),
                                 "dwd": (dy, None, h, eh)}.items():
        val, e = product(p.t(), q, None if ep is None else ep.t(), eq)
        out[name] = (val, e + up * (val.abs() + e))
    t = dy.shape[0]
    for name, p, ep in (("dbg", dg, edg), ("dbu", du, edu), ("dbd", dy, torch.zeros_like(dy))):
        val = p.sum(0)
        e = ep.sum(0) + (t + 2) * SUM * p.abs().sum(0)
        out[name] = (val, e + up * (val.abs() + e))
    return out


def check(name, got, want, bound, roundings, dtype):
    """Every element within its bound, and the whole within `roundings` roundings by norm."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - want).abs() - bound
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{name}: {float((got - want).abs().max()):.3e} off, over its bound by {float(over.max()):.3e}"
    norm = float(want.norm())
    if norm > 0:
        rel = float((got - want).norm()) / norm
        limit = roundings * U[dtype] if dtype == torch.bfloat16 else 1e-5
        assert rel <= limit, f"{name}: relative error {rel:.3e} > {limit:.3e}"
