"""Distillation from a teacher's top logits in 64 bits, with how far evaluations in 32 bits may be from it, for the tests."""
import math

import torch

from head_oracle import EPS32


def _softmax(x, tau):
    """(q, log q, relative bound of q, absolute bound of log q) over all classes.  A power of two is off by 2^-22 of itself and by its
    argument's two roundings; sums are chains of V / 256 + 80 additions, rescaled a dozen times at most."""
    d = (x - x.amax(1, keepdim=True)) / tau
    log_q = torch.log_softmax(x / tau, 1)
    q = log_q.exp()
    far = torch.where(q > 0, d.abs(), 0.0)
    rel_s = (x.size(1) / 256 + 80) * EPS32 + 12 * 2.0 ** -22 + 2.0 ** -22 * (q * far).sum(1, keepdim=True)
    log_s = (log_q - d).nan_to_num(0.0).abs().amax(1, keepdim=True)
    return q, log_q, rel_s + 2.0 ** -22 * (1 + far), rel_s + 2.0 ** -22 * (far + log_s)


def loss_and_gradient(x, values, indices, targets, tau, mix, up):
    """(losses, bound, dx, bound) of rows; up: a number per row."""
    x, values, up = x.double(), values.double(), up.double().view(-1, 1)
    rows, V = x.shape
    there = (indices >= 0) & (values > -math.inf)
    some = there.any(1, keepdim=True)
    at = indices.clamp_min(0)
    part = 1.0 - mix
    t = torch.where(there, values / tau, torch.where(some, -math.inf, 0.0))
    log_p = torch.log_softmax(t, 1)
    p = torch.where(there, log_p.exp(), 0.0)
    top = t.amax(1, keepdim=True)
    spread = torch.where(there, (t - top).abs() + t.abs() + top.abs(), 0.0)
    rel_p = 2.0 ** -21 * (1 + spread) + (values.size(1) / 32 + 8) * EPS32 + (p * 2.0 ** -21 * (1 + spread)).sum(1, keepdim=True)
    q, log_q, rel_q, off_log_q = _softmax(x, tau)
    term = torch.where(p > 0, log_p - torch.gather(log_q, 1, at), 0.0)
    losses = part * tau ** 2 * (p * term).sum(1)
    log_sum = (log_p - (t - top)).nan_to_num(0.0, neginf=0.0).abs().amax(1, keepdim=True)
    off = p * (torch.gather(off_log_q, 1, at) + 2.0 ** -21 * (spread + log_sum) + rel_p * term.nan_to_num(0.0).abs() + 8 * EPS32 * term.nan_to_num(0.0).abs())
    off_loss = part * tau ** 2 * torch.where(p > 0, off, 0.0).sum(1) + 8 * EPS32 * losses.abs()
    w = torch.where(some, up * part * tau, 0.0)
    dx = torch.where(some, w * q, 0.0)
    off_dx = dx.abs() * (rel_q + 8 * EPS32)
    take = w * p
    dx = dx.scatter_add(1, at, -take)
    off_dx = off_dx.scatter_add(1, at, take.abs() * (rel_p + (values.size(1) + 8) * EPS32))
    if mix:
        label = (targets >= 0).view(-1, 1)
        target = targets.clamp_min(0).view(-1, 1)
        q, log_q, rel_q, off_log_q = _softmax(x, 1.0)
        losses = losses - mix * torch.where(label, torch.gather(log_q, 1, target), 0.0).view(-1)
        off_loss = off_loss + mix * torch.where(label, torch.gather(off_log_q, 1, target), 0.0).view(-1) + 8 * EPS32 * losses.abs()
        w = torch.where(label, up * mix, 0.0)
        more = torch.where(label, w * q, 0.0)
        dx = dx + more
        dx = dx.scatter_add(1, target, -w)
        off_dx = off_dx + more.abs() * (rel_q + 8 * EPS32) + 4 * EPS32 * dx.abs()
        off_dx = off_dx.scatter_add(1, target, 4 * EPS32 * w.abs())
    return losses, off_loss, dx, off_dx
