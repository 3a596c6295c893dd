"""The layers' formulas in 64 bits, and how far the kernels may be from them.

A rounding to a type is off by at most u = eps / 2 of the value.  The kernels add products of exact operands in fp32, in some order: the sum
is off by at most terms * 2^-24 of the sum of magnitudes (+ 4 for bias, join and residual).  An activation is evaluated in fp32 within 2^-20 of
max(1, |z|) (a handful of operations and math functions of a few steps each) and carries an error of z on with a slope of at most 1.2; so does
its derivative, whose slope is at most 1.2 too and which is at most 1.2 itself.  What is kept for the backward pass is cut off behind 16 bits of
the significand (2^-15 at most, bf16 tensors) or kept whole, and its product with the incoming gradient is rounded."""
import math

import torch

F32 = 2.0 ** -24


def cut(dtype):
    return 2.0 ** -15 if dtype == torch.bfloat16 else 0.0


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def activation(name, z):
    """(act(z), act'(z)) for float64 z."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z), (~(z <= 0)).double()
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return (s, s * (1 - s)) if name == "sigmoid" else (z * s, s * (1 + z * (1 - s)))


def product(x, w, b):
    """x w^T + b and the bound of its fp32 sum."""
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b, mag + b.abs()
    return z, (x.size(1) + 4) * F32 * mag


def activated(name, z, ez):
    """act(z), act'(z) and their bounds (relu: act' is exact where the sum cannot change its sign)."""
    a, d = activation(name, z)
    if name == "none":
        return a, d, ez, torch.zeros_like(z)
    ev = 2.0 ** -20 * z.abs().clamp_min(1.0)
    if name == "relu":
        return a, d, ez, (z.abs() <= ez).double()
    return a, d, 1.2 * ez + ev, 1.2 * ez + ev


def linear(x, w, b, r, name, dy, dtype):
    """{name: (value, bound)} of the result and every gradient."""
    u = unit(dtype)
    x, w, b, r, dy = (None if t is None else t.detach().double() for t in (x, w, b, r, dy))
    z, ez = product(x, w, b)
    a, d, ea, ed = activated(name, z, ez)
    y = a if r is None else a + r
    out = {"y": (y, ea + (u + 2 * F32) * (y.abs() + ea))}
    dz = dy * d
    kept = 0.0 if name == "none" else cut(dtype)
    edz = dy.abs() * (ed + kept * (d.abs() + ed))          # of the unrounded product
    made = edz + (0.0 if name == "none" else u + F32) * (dz.abs() + edz)  # of the rounded one
    mag = dz.abs() + made
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    edx = made @ w.abs() + (w.size(0) + 4) * F32 * (mag @ w.abs())
    edw = made.t() @ x.abs() + (x.size(0) + 4) * F32 * (mag.t() @ x.abs())
    edb = edz.sum(0) + (x.size(0) + 4) * F32 * mag.sum(0)
    out["dx"] = (dx, edx + u * (dx.abs() + edx))
    out["dw"] = (dw, edw + u * (dw.abs() + edw))
    out["db"] = (db, edb + u * (db.abs() + edb))
    out["dr"] = (dy, torch.zeros_like(dy))
    return out


def gated(x, wg, wu, bg, bu, name, dh, dtype):
    u = unit(dtype)
    x, wg, wu, bg, bu, dh = (None if t is None else t.detach().double() for t in (x, wg, wu, bg, bu, dh))
    g, eg = product(x, wg, bg)
    v, ev = product(x, wu, bu)
    a, d, ea, ed = activated(name, g, eg)
    h = a * v
    eh = ea * v.abs() + a.abs() * ev + ea * ev + 2 * F32 * h.abs()
    out = {"y": (h, eh + u * (h.abs() + eh))}
    et = ed * v.abs() + d.abs() * ev + ed * ev + 2 * F32 * (d * v).abs()
    dzs = []
    for factor, ef in ((d * v, et), (a, ea)):  # of g, of u
        kept = ef + cut(dtype) * (factor.abs() + ef)
        dz = dh * factor
        edz = dh.abs() * kept + F32 * (dz.abs() + dh.abs() * kept)
        dzs.append((dz, edz, edz + (u + F32) * (dz.abs() + edz)))
    dx = sum(dz @ w for (dz, _, _), w in zip(dzs, (wg, wu)))
    edx = sum(m @ w.abs() + (2 * w.size(0) + 4) * F32 * ((dz.abs() + m) @ w.abs()) for (dz, _, m), w in zip(dzs, (wg, wu)))
    out["dx"] = (dx, edx + u * (dx.abs() + edx))
    for i, (dz, e, m) in enumerate(dzs):
        mag = dz.abs() + m
        dw, edw = dz.t() @ x, m.t() @ x.abs() + (x.size(0) + 4) * F32 * (mag.t() @ x.abs())
        db, edb = dz.sum(0), e.sum(0) + (x.size(0) + 4) * F32 * mag.sum(0)
        out[f"dw{i}"] = (dw, edw + u * (dw.abs() + edw))
        out[f"db{i}"] = (db, edb + u * (db.abs() + edb))
    return out


def check(name, got, want, bound):
    """Every value of `got` lies within its bound of the value wanted (where that is not finite, it is the same)."""
    got = got.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[~fine].nan_to_num(), want[~fine].nan_to_num()), name
    off = ((got - want).abs() - bound)[fine]
    # (a bound of zero is a value that is copied; 1e-37 stands for what underflows)
    assert not off.numel() or off.max().item() <= 1e-37, (name, off.max().item(), (got - want).abs()[fine].max().item())
