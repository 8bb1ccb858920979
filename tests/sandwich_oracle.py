"""The residual stream between two norms in 64 bits, with how far evaluations in 32 bits may be from it, for the tests."""
import torch

from head_oracle import EPS32, norm, norm_grad


def _or(p, value, x):
    return torch.full_like(x[:1, :].double(), value) if p is None else p.double()


def forward(x, residual, gate, scale, pw, pb, eps):
    """(h, bound) before h is rounded; y is head_oracle.norm of what is held."""
    n, _, _, _, off = norm(x, pw, pb, eps)
    by = _or(scale, 1.0, x) * (1.0 if gate is None else gate.double())
    h = residual.double() + by * n
    return h, by.abs() * off + 6 * EPS32 * ((by * n).abs() + h.abs())


def backward(dy, dh, x, h, gate, scale, pw, pb, w, eps):
    """{name: (gradient, bound)} given the h that is held; dy or dh may be None."""
    x64 = x.double()
    g = torch.ones_like(x64) if gate is None else gate.double().expand_as(x64)
    s, w1 = _or(scale, 1.0, x), _or(pw, 1.0, x)
    out = {}
    zero = torch.zeros_like(x64)
    (d, off_d), out["w"], out["b"] = norm_grad(zero if dy is None else dy, h, w, eps)
    if dh is not None:
        d = d + dh.double()
        off_d = off_d + 2 * EPS32 * d.abs()
    out["residual"] = d, off_d
    n, z, rstd, off_z, off_n = norm(x, pw, pb, eps)
    rows, C = x.shape
    dg = d * s * n
    off_dg = off_d * (s * n).abs() + (d * s).abs() * off_n + 6 * EPS32 * (d * s).abs() * (n.abs() + (z * w1).abs())
    if gate is not None:
        if gate.size(1) == 1 and C > 1:
            out["gate"] = dg.sum(1, keepdim=True), (off_dg + (C / 128 + 44) * EPS32 * (dg.abs() + off_dg)).sum(1, keepdim=True)
        else:
            out["gate"] = dg, off_dg
    # the sums P and Q, of which scale and the first norm's parameters have their gradients
    up = d * g
    off_up = off_d * g.abs() + 2 * EPS32 * up.abs()
    _, (P, off_P), (Q, off_Q) = norm_grad(up, x, None, eps)
    off_P, off_Q = off_P + (off_up * z.abs()).sum(0), off_Q + off_up.sum(0)
    b1 = _or(pb, 0.0, x)[0] if pb is None else pb.double()
    s1, w11 = (t[0] if t.dim() == 2 else t for t in (s, w1))
    out["pw"] = s1 * P, s1.abs() * off_P + 2 * EPS32 * (s1 * P).abs()
    out["pb"] = s1 * Q, s1.abs() * off_Q + 2 * EPS32 * (s1 * Q).abs()
    out["scale"] = w11 * P + b1 * Q, w11.abs() * off_P + b1.abs() * off_Q + 4 * EPS32 * ((w11 * P).abs() + (b1 * Q).abs())
    b = up * s
    off_b = off_up * s.abs() + 2 * EPS32 * b.abs()
    (gx, off_x), _, _ = norm_grad(b, x, pw, eps)
    through = off_b * w1.abs()
    out["x"] = gx, off_x + rstd * (through + through.mean(1, keepdim=True) + z.abs() * (through * z.abs()).mean(1, keepdim=True))
    return out
