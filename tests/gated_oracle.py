"""The gated projection in 64 bits with how far evaluations by the kernels may be from it, for the tests: plain tensor operations."""
import math

import torch

from head_oracle import EPS32, UNIT

# largest |act'| and |act''| (of the logistic function itself for "sigmoid")
SLOPE = {"silu": 1.1, "gelu": 1.13, "sigmoid": 0.25, "relu": 1.0}
CURVE = {"silu": 0.5, "gelu": 0.8, "sigmoid": 0.1, "relu": 0.0}


def act(g, name):
    """(act(g), act'(g))"""
    if name == "relu":
        return g.clamp_min(0), (g > 0).double()
    if name == "gelu":
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if name == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def sum_unit(terms, dtype):
    """How far a sum of `terms` products may be off, in units of the sum of their magnitudes.  Products of 16 bits: an instruction adds 16 of
    them to the accumulator and drops less than its last place, 2^-23.  Of 32 bits: 256 terms at a time (16 instructions with whole
    magnitudes and five times as many with 2^-8 of them at most: less than 24), then additions in 32 bits; 2^-26 of each product
    is left out.  A handful of rows: chains of terms / 128 additions and a dozen more."""
    if dtype == torch.float32:
        return 24 * 2.0 ** -23 + (terms / 128 + 16) * EPS32 + 2.0 ** -26
    return (terms / 16 + 16) * 2.0 ** -23


def forward(x, wg, wu, bg, bu, name, dtype):
    """dict: y, g, u in 64 bits, and how far g, u and (before it is rounded) y may be off."""
    x, wg, wu = x.double().flatten(0, -2), wg.double(), wu.double()
    out = {}
    for key, w, b in (("g", wg, bg), ("u", wu, bu)):
        v = x @ w.t()
        off = sum_unit(x.size(1), dtype) * (x.abs() @ w.abs().t())
        if b is not None:
            v = v + b.double()
            off = off + EPS32 * v.abs()
        out[key], out["off_" + key] = v, off
    a, _ = act(out["g"], name)
    out["y"] = a * out["u"]
    # (the functions: a few units of 32 bits of themselves; e^-g has a relative error of |g| units)
    off_a = SLOPE[name] * out["off_g"] + (8 + out["g"].abs()) * EPS32 * a.abs()
    out["off_y"] = off_a * (out["u"].abs() + out["off_u"]) + a.abs() * out["off_u"] + 2 * EPS32 * out["y"].abs()
    return out


def backward(dy, x, wg, wu, f, name, dtype):
    """{name: (gradient, bound)} before the last rounding."""
    unit = 0.0 if dtype == torch.float32 else UNIT[dtype]
    dy, x, wg, wu = dy.double().flatten(0, -2), x.double().flatten(0, -2), wg.double(), wu.double()
    a, s = act(f["g"], name)
    # (their gradients enter the products in the rows' type)
    off_g, off_u = f["off_g"] + EPS32 * f["g"].abs(), f["off_u"] + EPS32 * f["u"].abs()
    dg, du = dy * f["u"] * s, dy * a
    off_s = CURVE[name] * off_g + (16 + 4 * f["g"].abs()) * EPS32
    if name == "relu":  # (on the other side of zero)
        off_s = off_s + (f["g"].abs() <= f["off_g"]).double()
    off_dg = dy.abs() * (off_s * (f["u"].abs() + off_u) + s.abs() * off_u) + 4 * EPS32 * dg.abs()
    off_du = dy.abs() * (SLOPE[name] * off_g + (8 + f["g"].abs()) * EPS32 * a.abs()) + 4 * EPS32 * du.abs()
    out = {}
    chain = (dy.size(0) / 8 + 64) * EPS32
    for key, d, off in (("b_gate", dg, off_dg), ("b_up", du, off_du)):
        out[key] = d.sum(0), off.sum(0) + chain * d.abs().sum(0)
    sg, su = dg.abs() + off_dg, du.abs() + off_du
    off_dg, off_du = off_dg + unit * sg, off_du + unit * su
    for key, d, off, size in (("w_gate", dg, off_dg, sg), ("w_up", du, off_du, su)):
        out[key] = d.t() @ x, (off + sum_unit(x.size(0), dtype) * size).t() @ x.abs()
    n = sum_unit(2 * wg.size(0), dtype)
    out["x"] = dg @ wg + du @ wu, (off_dg + n * sg) @ wg.abs() + (off_du + n * su) @ wu.abs()
    return out
