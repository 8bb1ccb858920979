"""The head's operators in 64 bits (the generator in whole numbers), for the tests: plain tensor and array operations."""
import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}  # spacing of the smallest numbers
EPS32 = 2.0 ** -24


def philox(counter, key):
    """Philox4x32-10 of four arrays of words and two words."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k0, k1 = key
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        low, high = np.uint64(0xFFFFFFFF), np.uint64(32)
        c = [(b >> high) ^ c[1] ^ np.uint64(k0), b & low, (a >> high) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def words(n, seed, offset, first=0):
    """Words of the elements first .. first + n - 1."""
    i = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    c = philox([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)],
               (seed & 0xFFFFFFFF, seed >> 32))
    return np.stack(c, 1).reshape(-1)[first % 4:first % 4 + n]


def keep(shape, p, seed, offset):
    n = int(np.prod(shape))
    return torch.from_numpy((words(n, seed, offset) >= np.uint64(round(p * 2 ** 32))).reshape(shape)) if p < 1 else \
        torch.zeros(shape, dtype=torch.bool)


def dropped(x, kept, p):
    """In 32 bits, as the operator is defined: the product with 1 / (1 - p) rounded by itself."""
    scale = float(np.float32(1.0 / (1.0 - p))) if p < 1 else 0.0
    return torch.where(kept.to(x.device), x.float() * torch.tensor(scale, device=x.device), torch.zeros((), device=x.device))


def norm(x, weight, bias, eps):
    """(y, z, 1 / deviation, bound) in 64 bits; bound: how far an evaluation in 32 bits may be from y before it is rounded."""
    x = x.double()
    C = x.size(-1)
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    z = (x - mean) * rstd
    w = torch.ones_like(x[..., :1]) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    y = z * w + b
    # sums of C terms with chains of at most C / 128 + 32 additions: the mean is off by that many units of the mean magnitude,
    # the deviation by as many of itself and by what the mean's error takes along; a dozen roundings more around them
    chain = (C / 128 + 44) * EPS32
    off_z = chain * (z.abs() + 2 * rstd * x.abs().mean(-1, keepdim=True))
    return y, z, rstd, off_z, off_z * w.abs() + 4 * EPS32 * (y.abs() + b.abs())


def near(got, want, bound):
    """Every element of `got` is the rounding of a number within `bound` of `want`."""
    d = (got.double() - want).abs()
    limit = bound + (want.abs() + bound) * UNIT[got.dtype] + LEAST[got.dtype]
    return bool((d <= limit).all())


def norm_grad(grad, x, weight, eps):
    """(grad_x, grad_weight, grad_bias) in 64 bits and how far evaluations in 32 bits may be from them."""
    y, z, rstd, off_z, _ = norm(x, weight, None, eps)
    g = grad.double()
    a = g if weight is None else g * weight.double()
    m1, m2 = a.mean(-1, keepdim=True), (a * z).mean(-1, keepdim=True)
    gx = rstd * (a - m1 - z * m2)
    rows, C = x.numel() // x.size(-1), x.size(-1)
    chain = (C / 128 + 48) * EPS32
    size = a.abs() + a.abs().mean(-1, keepdim=True) + z.abs() * (a * z).abs().mean(-1, keepdim=True)
    off_z2 = (a.abs() * off_z).mean(-1, keepdim=True)
    # (the deviation's own error is that of z as a whole, relative)
    off_x = rstd * (2 * chain * size + off_z * (a * z).abs().mean(-1, keepdim=True) + z.abs() * off_z2) + \
        gx.abs() * (off_z.amax(-1, keepdim=True) / z.abs().amax(-1, keepdim=True).clamp_min(1e-30)).clamp_max(1.0)
    flat = lambda t: t.reshape(rows, C)  # noqa: E731
    column = (rows / 4 + 64) * EPS32
    gw, gb = flat(g * z).sum(0), flat(g).sum(0)
    off_w = column * flat(g * z).abs().sum(0) + flat(g.abs() * off_z).sum(0)
    return (gx, off_x), (gw, off_w), (gb, column * flat(g).abs().sum(0))


def quantise(x):
    """(q, scale) by the operator's definition, in 32 bits on the host."""
    x = x.detach().float().cpu().numpy()
    with np.errstate(all="ignore"):
        scale = np.abs(x).max(-1) / np.float32(127)
        scale = np.where(scale < np.float32(2.0 ** -126), np.float32(2.0 ** -126), scale)
        q = np.rint(x * (np.float32(1) / scale)[..., None])
    return torch.from_numpy(q), torch.from_numpy(scale)


def product(q, scale, wq, w_scale, bias, activation):
    """(y, bound) in 64 bits from the integers."""
    y = q.double() @ wq.double().t() * scale.double().unsqueeze(-1) * w_scale.double()
    bound = 4 * EPS32 * y.abs()
    if bias is not None:
        y = y + bias.double()
        bound = bound + EPS32 * y.abs()
    if activation == "relu":
        y = y.relu()
    if activation == "tanh":
        bound = bound * (1 - y.tanh() ** 2 + 1e-6) + 4 * EPS32
        y = y.tanh()
    return y, bound
