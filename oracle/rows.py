"""64-bit CPU definitions of the row operators (LayerNorm, the 8-bit kept form, the sigmoid gate, 8-bit
integer rows), each with how far a float32 computation rounded once to the output's type may be from it.

A rounding to type T is off by at most half a step, eps(T) / 2 of the value; u = 2^-24 for float32. A sum over a
row passes at most 8 roundings in a thread, or 16 where a warp has the row alone, one between the thread's
two halves, 5 over the warp and 32 over a block's warps: at most SUM = 46, relative to the sum of magnitudes.
"""
import math

import torch

U = 2.0 ** -24
SUM = 46
BLOCK = 128


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half the smallest spacing of the type: what a value near zero may be off by."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def kept(x):
    """(what the kept form of x [..., D] stands for, unit of each element, share of a unit to the nearest tie)."""
    x = x.double()
    out, units, ties = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    for at in range(0, x.shape[-1], BLOCK):
        part = x[..., at:at + BLOCK]
        a = part.abs().amax(-1, keepdim=True)
        e = torch.frexp(a / 127.5)[1].double().clamp(min=-126)  # smallest e with 2^e > a / 127.5
        unit = torch.exp2(e)
        top = torch.where(e >= 122, 63.0, 127.0)
        code = torch.round(part / unit).clamp(-top, top)
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        out[..., at:at + BLOCK] = torch.where(bad, math.nan, code * unit)
        units[..., at:at + BLOCK] = unit.expand_as(part)
        frac = part / unit - torch.floor(part / unit)
        # where the block's largest magnitude is near a border, its unit may come out twice or half
        near = (torch.frexp(a / 127.5)[0] - 0.5).abs().clamp(max=1) < 1e-5
        near = near | ((torch.frexp(a / 127.5)[0] - 1.0).abs() < 1e-5)
        ties[..., at:at + BLOCK] = torch.where(near.expand_as(part), 0.0, (frac - 0.5).abs())
    return out, units, ties


def layer_norm(x, w, b, eps, dtype):
    """y, its error bound, and for the backward (h, 1/sigma, error bound of h)."""
    x = x.double()
    w = torch.ones_like(x) if w is None else _over(w, x)
    b = torch.zeros_like(x) if b is None else _over(b, x)
    mean = x.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - mean) * rs
    top = x.abs().amax(-1, keepdim=True)
    # the mean: SUM + 2 roundings of values up to top; the variance's relative error: (SUM + 4) u plus twice
    # the relative error of the centred values, half of it in 1/sigma, and three roundings
    dh = U * ((SUM + 4) * top * rs + (SUM / 2 + 8) * h.abs() + (SUM + 4) * top * rs * h.abs())
    y = h * w + b
    tol = half_step(dtype) * y.abs() + w.abs() * dh + 2 * U * ((h * w).abs() + b.abs()) + floor_of(dtype)
    return y, tol * (1 + 1e-3), (h, rs, dh)


def _over(w, x):
    w = w.double()
    return (w if w.ndim == 1 else w.reshape(w.shape[0], *(1,) * (x.ndim - 2), w.shape[1])).expand_as(x)


def layer_norm_backward(h, rs, dh, w, dy, dtype, wdtype, keep8=False, groups=None):
    """(dx, tol), (dw, tol), (db, tol); groups: the shape of w, [D] or [G, D]."""
    dy = dy.double()
    wx = torch.ones_like(dy) if w is None else _over(w, dy)
    if keep8:
        h, unit, tie = kept(h)
        dh = torch.where(tie <= dh / unit + 1e-9, unit + 1e-12, 0.0)  # another code, by one unit
    gw = dy * wx
    s1, s2 = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
    d1 = U * (SUM + 3) * gw.abs().mean(-1, keepdim=True)
    d2 = U * (SUM + 4) * (gw * h).abs().mean(-1, keepdim=True) + (gw.abs() * dh).mean(-1, keepdim=True)
    dx = rs * (gw - s1 - h * s2)
    rel = U * (SUM + 20)
    # (h + dh)(s2 + d2) - h s2, and the roundings of the three terms
    tol = rs * (d1 + (h.abs() + dh) * d2 + s2.abs() * dh + 4 * U * (gw.abs() + s1.abs() + (h * s2).abs())) + rel * dx.abs()
    # 1/sigma carries the error of the centred values' second moment
    tol = tol * (1 + 1e-3) + half_step(dtype) * dx.abs() + floor_of(dtype)
    shape = groups or (dy.shape[-1],)
    rows = (lambda t: t.reshape(-1, t.shape[-1]).sum(0)) if len(shape) == 1 else \
        (lambda t: t.reshape(shape[0], -1, t.shape[-1]).sum(1))
    n = dy.numel() // dy.shape[-1] // (shape[0] if len(shape) == 2 else 1)
    dw, db = rows(dy * h), rows(dy)
    tw = (n + 2) * U * rows((dy * h).abs()) + rows(dy.abs() * dh) + half_step(wdtype) * dw.abs() + floor_of(wdtype)
    tb = (n + 2) * U * rows(dy.abs()) + half_step(wdtype) * db.abs() + floor_of(wdtype)
    return (dx, tol), (dw, tw), (db, tb)


def gate(x, z, dtype):
    """y and its bound. 32-bit gates: expf and divisions, 8 u; 16-bit: the fast exponential's
    2 + 1.2 |z| units of 2^-23, the fast division's 2, and the sums'."""
    x, z = x.double(), z.double()
    rel = gate_error(z, dtype)
    y = x * torch.sigmoid(z)
    return y, (half_step(dtype) + rel + U) * y.abs() + floor_of(dtype)


def gate_error(z, dtype):
    return 8 * U + 0 * z if dtype == torch.float32 else (8 + 1.2 * z.abs().clamp(max=80)) * 2 * U


def gate_backward(x, z, dy, dtype, keep8=False):
    if keep8:
        x, z = kept(x)[0], kept(z)[0]
    x, z, dy = x.double(), z.double(), dy.double()
    rel = gate_error(z, dtype)
    dx = dy * torch.sigmoid(z)
    dz = dy * x * torch.sigmoid(z) * torch.sigmoid(-z)
    return ((dx, (half_step(dtype) + rel + U) * dx.abs() + floor_of(dtype)),
            (dz, (half_step(dtype) + 2 * rel + 3 * U) * dz.abs() + floor_of(dtype)))


def int8_rows(x):
    """(codes as float64, scale float32) by the definition's own float32 steps, which IEEE arithmetic fixes."""
    x = x.float()
    a = x.abs().amax(-1, keepdim=True) if x.shape[-1] else x.new_zeros((*x.shape[:-1], 1))
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    small = a < 2.0 ** -118
    f = torch.where(bad | small, torch.zeros_like(a), torch.tensor(127.0) / a)
    codes = torch.round(torch.where(f == 0, torch.zeros_like(x), x) * f)
    return codes.double(), torch.where(bad, torch.full_like(a, math.nan), a / 127)[..., 0]


def int8_product(codes, scale, w_codes, w_scale, bias, dtype):
    """The product of integer rows and its bound: the integer sum's rounding to float32, two products and
    the addition, then the type's."""
    prod = (codes.double() @ w_codes.double().t()) * scale.double()[..., None] * w_scale.double()
    b = torch.zeros(w_codes.shape[0], dtype=torch.float64) if bias is None else bias.double()
    out = prod + b
    return out, half_step(dtype) * out.abs() + 4 * U * prod.abs() + 2 * U * out.abs() + floor_of(dtype)
