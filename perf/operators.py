"""What is followed of the head's operators: layer norm, dropout, both joined on a residual stream, and the product in 8-bit integers.

They stand behind the distance layers of a network: a residual feed-forward head is trained with `layer_norm`, `dropout` and
`dropout_add_layer_norm`, and answers with `layer_norm_quantized` and `int8_linear`.  A case is a dict of plain values; `call` says
what the user's program calls:

  norm     layer_norm of `rows` rows of `C`: forward, and with `grad` the gradients of the rows, the weight and the bias
  dropout  dropout of rows x C (onto a residual where `residual`), forward and the gradient
  join     dropout_add_layer_norm: h = residual + dropout(x), y = layer norm of h, forward and all gradients
  linear   int8_linear of `M` tokens, K -> N, the tokens in floating point (quantised in the call)
  serve    layer_norm_quantized, int8_linear K -> N with ReLU, int8_linear N -> K: a head's block as it answers

`type` is that of the activations ("f32", "f16", "bf16"); `params` that of the norm's weight and bias.  Rows whose `pitch` is not C
are slices of wider ones.  Activations are N(0, 1) with a scale and a mean of their own per row, as behind distance layers;
upstream gradients are N(0, 1); weights are 1 + N(0, 0.1) in a norm and N(0, 1 / K) in a product, quantised beforehand
per output channel, in rows that start at multiples of 16 bytes.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
LEAST_SCALE = 2.0 ** -126  # of a quantised row


def listed():
    return [
        # a training batch of an MNIST network of width 1024: launches count
        dict(name="norm-small-train", call="norm", rows=64, C=1024, type="f32", params="f32", grad=True),
        # the widest hidden layer, a global batch on one card, mixed precision
        dict(name="norm-wide-train", call="norm", rows=16384, C=5120, type="bf16", params="f32", grad=True),
        # the positions of a convolution's 32 x 32 images: many short rows
        dict(name="norm-positions-train", call="norm", rows=131072, C=96, type="bf16", params="bf16", grad=True),
        # rows of odd length in an evaluation, no parameters
        dict(name="norm-ragged-eval", call="norm", rows=9999, C=1001, type="f16", params="none", grad=False),
        # hidden activations of a training batch
        dict(name="dropout-hidden", call="dropout", rows=512, C=5120, type="f32", p=0.1, residual=False),
        # rows of odd length, the largest batch
        dict(name="dropout-ragged-large", call="dropout", rows=16383, C=4097, type="bf16", p=0.25, residual=True),
        # the residual stream of a head in a small batch
        dict(name="join-small", call="join", rows=128, C=512, type="f32", params="f32", p=0.1),
        # the same at the widest, a large batch
        dict(name="join-wide", call="join", rows=8192, C=5120, type="bf16", params="f32", p=0.1),
        # one image answered: the weight's bytes count
        dict(name="linear-single", call="linear", M=1, N=5120, K=5120, type="bf16", bias=True, act="none"),
        # the first layer of the hybrid model's head, a rank's batch, odd row length
        dict(name="linear-head", call="linear", M=64, N=512, K=5119, type="f32", bias=True, act="tanh"),
        # a whole test set in one call
        dict(name="linear-test-set", call="linear", M=10000, N=5120, K=5120, type="bf16", bias=False, act="none"),
        # a block of a head that answers a batch
        dict(name="serve-batch", call="serve", M=512, N=2048, K=5120, type="bf16", params="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["norm", "norm", "dropout", "join", "linear", "linear", "serve"])
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    if call in ("linear", "serve"):
        case = dict(call=call, M=_log(rng, 1, 10000), N=_log(rng, 10, 5120), K=_log(rng, 100, 8192), type=kind)
        if call == "linear":
            case.update(bias=rng.random() < 0.5, act=rng.choice(["none", "none", "relu", "tanh"]))
        else:
            # (a block's answers have 16 bits: in 32 the rounding of the norm decides between neighbouring integers)
            case.update(type=rng.choice(["f16", "bf16"]), N=_log(rng, 100, 5120), params=rng.choice(["f32", "same"]))
    else:
        case = dict(call=call, rows=_log(rng, 1, 131072), C=_log(rng, 10, 16384), type=kind)
        if call == "norm":
            case.update(params=rng.choice(["f32", "f32", "same", "none"]), grad=rng.random() < 0.7)
            if rng.random() < 0.2:
                case["pitch"] = case["C"] + rng.choice([1, 8, 64])
        else:
            case["p"] = round(rng.uniform(0.02, 0.6), 3)
            case.update(dict(residual=rng.random() < 0.5) if call == "dropout" else dict(params=rng.choice(["f32", "f32", "same"])))
    if case.get("params") == "same":
        case["params"] = case["type"]
    rows = "M" if "M" in case else "rows"
    most = [c for c in listed() if c["call"] == call]
    while any(work(case)[w] > max(work(c)[w] for c in (most if w == "bytes" and rows == "rows" else listed())) for w in ("bytes", "flops")):
        case[rows] = max(1, case[rows] // 2)
        if case[rows] == 1:
            break
    return case


def _pitch(k):
    return (k + 15) // 16 * 16


def work(case):
    size = SIZES[case["type"]]
    if case["call"] in ("linear", "serve"):
        M, N, K = case["M"], case["N"], case["K"]
        if case["call"] == "linear":
            return dict(bytes=size * M * (K + N) + N * K + 4 * N * (2 if case["bias"] else 1), flops=2 * M * N * K)
        return dict(bytes=size * M * 2 * K + 2 * N * K + 8 * (N + K) + 2 * K * SIZES[case["params"]], flops=4 * M * N * K)
    n, C = case["rows"] * case["C"], case["C"]
    param = 0 if case.get("params", "none") == "none" else C * SIZES[case["params"]]
    if case["call"] == "norm":
        return dict(bytes=(4 if case["grad"] else 2) * n * size + (4 if case["grad"] else 2) * param, flops=(20 if case["grad"] else 8) * n)
    if case["call"] == "dropout":  # (x, out, gradient in, gradient out [, residual]; about 20 operations per word)
        return dict(bytes=(4 + bool(case["residual"])) * n * size, flops=44 * n)
    return dict(bytes=8 * n * size + 4 * param, flops=66 * n)


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _activations(rows, C, kind, f, pitch=None):
    x = torch.randn(rows, pitch or C, **f)
    x.mul_(torch.rand(rows, 1, **f).mul_(2).add_(0.5)).add_(torch.randn(rows, 1, **f))
    x = x.to(TYPES[kind])
    return x if pitch is None else x[:, :C]


def _quantised_weight(N, K, f):
    """Rows of 8-bit integers with a scale per row, as a program keeps them."""
    w = torch.randn(N, K, **f) / math.sqrt(K)
    scale = w.abs().amax(1) / torch.full((N,), 127.0, device="cuda")
    q = torch.zeros(N, _pitch(K), device="cuda", dtype=torch.int8)[:, :K]
    q.copy_(torch.round(w / scale[:, None]))
    return q, scale


def prepare(case, seed):
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    s = dict(case=case, dtype=TYPES[case["type"]], seed=(seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63), offset=seed * 3 + 1)
    if case["call"] in ("linear", "serve"):
        M, N, K = case["M"], case["N"], case["K"]
        s.update(x=_activations(M, K, case["type"], f), weight=_quantised_weight(N, K, f), bias=None, weight2=None)
        if case["call"] == "serve" or case["bias"]:
            s["bias"] = torch.randn(N, **f)
        if case["call"] == "serve":
            s.update(weight2=_quantised_weight(K, N, f), bias2=torch.randn(K, **f))
        C = K
    else:
        rows, C = case["rows"], case["C"]
        s["x"] = _activations(rows, C, case["type"], f, case.get("pitch"))
        for name in ["dy"] * (case["call"] != "norm" or case["grad"]) + ["dh"] * (case["call"] == "join"):
            s[name] = torch.randn(rows, C, **f).to(s["dtype"])
        if case["call"] == "join" or case.get("residual"):
            s["residual"] = _activations(rows, C, case["type"], f)
    s["gamma"] = s["beta"] = None
    if case.get("params", "none") != "none":
        s["gamma"] = (1 + 0.1 * torch.randn(C, **f)).to(TYPES[case["params"]])
        s["beta"] = (0.1 * torch.randn(C, **f)).to(TYPES[case["params"]])
    for name in ("x", "residual", "gamma", "beta"):
        if s.get(name) is not None and "dy" in s:
            s[name] = s[name].detach().requires_grad_()
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------------
def _mulhilo(c, a):
    """High and low 32 bits of the product of the words `c` (held in 64 bits) and the constant `a`."""
    low, high = c & 0xFFFF, c >> 16
    t = (low * a >> 16) + high * a  # (below 2^49)
    return t >> 16, ((t & 0xFFFF) << 16) | (low * a & 0xFFFF)


def _words(n, seed, offset):
    """Words 0 .. n - 1 of Philox4x32 with 10 rounds: key `seed`, counter (block, offset), four words per block."""
    block = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1 = block & 0xFFFFFFFF, block >> 32
    c2, c3 = torch.full_like(block, offset & 0xFFFFFFFF), torch.full_like(block, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _plain_keep(s):
    c = s["case"]
    return (_words(c["rows"] * c["C"], s["seed"], s["offset"]) >= round(c["p"] * 2 ** 32)).view(c["rows"], c["C"])


def _plain_drop(v, keep, p):
    return torch.where(keep, v.float() * (1.0 / (1.0 - p)), 0.0)


def _plain_normed(x, gamma, beta):
    """(y in 32 bits, normalised rows, 1 / deviation) of rows in 32 bits."""
    d = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * rstd
    return (xh if gamma is None else xh * gamma.float() + beta.float()), xh, rstd


def _plain_norm_grad(dy, gamma, xh, rstd):
    """(dx, dgamma, dbeta) in 32 bits."""
    dy = dy.float()
    a = dy if gamma is None else dy * gamma.float()
    dx = rstd * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def _plain_quantise(x):
    scale = x.abs().amax(1) / torch.full((x.size(0),), 127.0, device=x.device)
    scale = scale.clamp_min(LEAST_SCALE)
    return torch.round(x * (1.0 / scale)[:, None]), scale


def _plain_product(q, scale, weight, bias, act):
    wq, ws = weight
    y = (q @ wq.float().t()) * scale[:, None] * ws
    if bias is not None:
        y = y + bias
    return torch.relu(y) if act == "relu" else torch.tanh(y) if act == "tanh" else y


def _plain(s):
    c, t, x = s["case"], s["dtype"], s["x"].detach().float()
    if c["call"] == "linear":
        return dict(y=_plain_product(*_plain_quantise(x), s["weight"], s["bias"], c["act"]).to(t))
    if c["call"] == "serve":
        u = _plain_product(*_plain_quantise(_plain_normed(x, s["gamma"], s["beta"])[0]), s["weight"], s["bias"], "relu").to(t)
        return dict(y=_plain_product(*_plain_quantise(u.float()), s["weight2"], s["bias2"], "none").to(t))
    if c["call"] == "norm":
        y, xh, rstd = _plain_normed(x, s["gamma"], s["beta"])
        if not c["grad"]:
            return dict(y=y.to(t))
        dx, dg, db = _plain_norm_grad(s["dy"], s["gamma"], xh, rstd)
        out = dict(y=y.to(t), dx=dx.to(t))
        return out if s["gamma"] is None else dict(out, dgamma=dg.to(s["gamma"].dtype), dbeta=db.to(s["gamma"].dtype))
    keep = _plain_keep(s)
    if c["call"] == "dropout":
        out = _plain_drop(x, keep, c["p"])
        if c["residual"]:
            out = s["residual"].detach().float() + out
        return dict(out=out.to(t), dx=_plain_drop(s["dy"], keep, c["p"]).to(t))
    # the residual stream is held in its type, and that is what is normalised
    h = (s["residual"].detach().float() + _plain_drop(x, keep, c["p"])).to(t)
    y, xh, rstd = _plain_normed(h.float(), s["gamma"], s["beta"])
    dx, dg, db = _plain_norm_grad(s["dy"], s["gamma"], xh, rstd)
    dres = dx + s["dh"].float()
    return dict(y=y.to(t), h=h, dx=_plain_drop(dres, keep, c["p"]).to(t), dresidual=dres.to(t), dgamma=dg.to(s["gamma"].dtype),
                dbeta=db.to(s["gamma"].dtype))


# ---- the framework's operators ----------------------------------------------------------------------------------------------------
def _framework(s):
    import l_inf_dist_net_v2_b200 as ldn
    c, x = s["case"], s["x"]
    if c["call"] == "linear":
        return dict(y=ldn.int8_linear(x, s["weight"], s["bias"], activation=c["act"]))
    if c["call"] == "serve":
        normed = ldn.layer_norm_quantized(x, s["gamma"], s["beta"], EPS)
        u = ldn.int8_linear(normed, s["weight"], s["bias"], activation="relu", out_dtype=s["dtype"])
        return dict(y=ldn.int8_linear(u, s["weight2"], s["bias2"]))
    if c["call"] == "norm":
        y = ldn.layer_norm(x, s["gamma"], s["beta"], EPS)
        if not c["grad"]:
            return dict(y=y)
        wanted = [x] if s["gamma"] is None else [x, s["gamma"], s["beta"]]
        return dict(zip(["y", "dx", "dgamma", "dbeta"], (y.detach(),) + torch.autograd.grad(y, wanted, s["dy"])))
    if c["call"] == "dropout":
        out = ldn.dropout(x, c["p"], s["seed"], s["offset"], residual=s.get("residual"))
        return dict(out=out.detach(), dx=torch.autograd.grad(out, x, s["dy"])[0])
    y, h = ldn.dropout_add_layer_norm(x, s["residual"], s["gamma"], s["beta"], c["p"], s["seed"], s["offset"], EPS)
    grads = torch.autograd.grad((y, h), (x, s["residual"], s["gamma"], s["beta"]), (s["dy"], s["dh"]))
    return dict(zip(["y", "h", "dx", "dresidual", "dgamma", "dbeta"], (y.detach(), h.detach()) + grads))


def run(state):
    if own:
        return _framework(state)
    with torch.no_grad():
        return _plain(state)


# ---- 64 bits --------------------------------------------------------------------------------------------------------------------
def _exact_keep(rows, C, seed, offset, p):
    """The kept elements, from the generator's definition in unsigned 64-bit arithmetic on the host."""
    n, m = rows * C, np.uint64(0xFFFFFFFF)
    counter = np.zeros((4, (n + 3) // 4), dtype=np.uint64)
    counter[0] = np.arange(counter.shape[1], dtype=np.uint64) & m
    counter[1] = np.arange(counter.shape[1], dtype=np.uint64) >> np.uint64(32)
    counter[2], counter[3] = offset % 2 ** 32, offset // 2 ** 32
    for r in range(10):
        key = [(seed + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32]
        a, b = counter[0] * np.uint64(0xD2511F53), counter[2] * np.uint64(0xCD9E8D57)
        counter = np.stack([(b >> np.uint64(32)) ^ counter[1] ^ np.uint64(key[0]), b & m,
                            (a >> np.uint64(32)) ^ counter[3] ^ np.uint64(key[1]), a & m])
    words = np.ascontiguousarray(counter.T).reshape(-1)[:n].reshape(rows, C)
    return torch.from_numpy(words >= np.uint64(round(p * 2 ** 32))).cuda()


def _exact_quantise(x):
    """The integers that the definition gives, whose scale is a number of 32 bits, and the scale."""
    x = x.float().cpu().numpy()
    scale = np.maximum(np.abs(x).max(1) / np.float32(127), np.float32(LEAST_SCALE)).astype(np.float32)
    q = np.rint(x * (np.float32(1) / scale)[:, None])
    return torch.from_numpy(q).cuda().double(), torch.from_numpy(scale).cuda().double()


def _exact_product(x, weight, bias, act):
    q, scale = _exact_quantise(x)
    y = torch.einsum("mk,nk->mn", q, weight[0].double()) * scale.view(-1, 1) * weight[1].double().view(1, -1)
    y = y if bias is None else y + bias.double().view(1, -1)
    return {"none": y, "relu": y.clamp_min(0), "tanh": y.tanh()}[act]


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    x, dtype = d["x"], s["dtype"]
    if case["call"] == "linear":
        return dict(y=_exact_product(s["x"], s["weight"], s["bias"], case["act"]))
    keep = None
    if case["call"] in ("dropout", "join"):
        keep = _exact_keep(case["rows"], case["C"], s["seed"], s["offset"], case["p"]).double() / (1 - case["p"])
        if case["call"] == "dropout":
            return dict(out=x * keep + d.get("residual", 0), dx=d["dy"] * keep)
        h = (x * keep + d["residual"]).to(dtype)
        x = h.double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sigma = (var + EPS).sqrt()
    g = d["gamma"] if "gamma" in d else torch.ones_like(x[0])
    y = (x - mean) / sigma * g + d.get("beta", 0)
    if case["call"] == "serve":
        u = _exact_product(y, s["weight"], s["bias"], "relu").to(dtype)
        return dict(y=_exact_product(u, s["weight2"], s["bias2"], "none"))
    out = dict(y=y)
    if "dy" not in d:
        return out
    # the gradient as the projection of dy g / sigma off the constant and off the normalised row
    a, z = d["dy"] * g / sigma, (x - mean) / sigma
    dx = a - a.mean(1, keepdim=True) - z * ((a * z).sum(1, keepdim=True) / x.size(1))
    if case["call"] == "join":
        out.update(h=d["residual"] + d["x"] * keep, dx=(dx + d["dh"]) * keep, dresidual=dx + d["dh"])
    else:
        out.update(dx=dx)
    if "gamma" in d:
        out.update(dgamma=(d["dy"] * z).sum(0), dbeta=d["dy"].sum(0))
    return out
