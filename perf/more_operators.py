"""What is followed of a gated residual head and the loss that it is distilled with.

The head stands behind the distance layers of a network.  Its blocks widen a row by two projections of which one gates the other
(`gated_linear`), and join the residual stream between two norms (`sandwich_norm`): one behind the block, whose rows a gate and a
scale weigh, and the next block's.  It is trained against the top logits of a larger teacher (`distillation_loss`).  A case is a dict
of plain values; `call` says what the user's program calls:

  gated     gated_linear of T rows, K -> H: act(x Wg' + bg) (x Wu' + bu), and with `grad` the gradients of rows, weights and biases
  sandwich  sandwich_norm of `rows` rows of `C`: h = residual + gate scale norm(x), y = norm(h), and with `grad` all gradients;
            `gate` is "none", "row" (one number per row) or "all" (one per element)
  distil    distillation_loss of `rows` rows of `V` logits against `k` of a teacher's, and its gradient; `labels`: mixed with the
            cross-entropy of labels; `ragged`: lists of different lengths, some empty, some rows without a label; `masked`: classes
            that are no choice have logits of minus infinity; `per_row`: a loss per row, and not the mean

`type` is that of the activations ("f32", "f16", "bf16"), of the projections' weights, and of the student's and the teacher's
logits; `params` that of the norms' parameters and the projections' biases.  Activations are N(0, 1) with a scale and a mean of
their own per row, as behind distance layers; rows of gated_linear have been through a norm and are N(0, 1).
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ["silu", "gelu", "sigmoid", "relu"]


def listed():
    return [
        # one image answered: the weights' bytes count
        dict(name="gated-single", call="gated", T=1, K=5120, H=5120, type="bf16", params="f32", bias=True, act="silu", grad=False),
        # a rank's batch answered by the hybrid model's head, odd row length
        dict(name="gated-ragged-eval", call="gated", T=64, K=5119, H=513, type="f16", params="f16", bias=True, act="gelu", grad=False),
        # a training step of the reference's batch, in its type
        dict(name="gated-batch-train", call="gated", T=512, K=5120, H=2048, type="f32", params="f32", bias=True, act="silu", grad=True),
        # the largest global batch on one card, mixed precision
        dict(name="gated-wide-train", call="gated", T=16384, K=5120, H=5120, type="bf16", params="bf16", bias=False, act="silu", grad=True),
        # a training batch of an MNIST network of width 1024: launches count
        dict(name="sandwich-small-train", call="sandwich", rows=64, C=1024, type="f32", params="f32", gate="row", grad=True),
        # the widest hidden layer, a global batch on one card, a gate of its own for each element
        dict(name="sandwich-wide-train", call="sandwich", rows=16384, C=5120, type="bf16", params="bf16", gate="all", grad=True),
        # the positions of a convolution's 32 x 32 images: many short rows
        dict(name="sandwich-positions-train", call="sandwich", rows=131072, C=96, type="bf16", params="bf16", gate="row", grad=True),
        # rows of odd length in an evaluation
        dict(name="sandwich-ragged-eval", call="sandwich", rows=9999, C=1001, type="f16", params="f32", gate="none", grad=False),
        # a batch of the ten classes: latency
        dict(name="distil-ten-classes", call="distil", rows=512, V=10, k=3, type="f32", tau=4.0, labels=True, ragged=False, masked=False, per_row=False),
        # a batch of a thousand classes
        dict(name="distil-thousand", call="distil", rows=8192, V=1000, k=20, type="f32", tau=2.0, labels=True, ragged=True, masked=False, per_row=True),
        # many classes, odd row length, some of them no choice
        dict(name="distil-ragged-large", call="distil", rows=8192, V=40001, k=64, type="bf16", tau=1.0, labels=True, ragged=True, masked=True, per_row=False),
        # few rows of very many classes
        dict(name="distil-few-rows", call="distil", rows=16, V=131072, k=100, type="bf16", tau=2.0, labels=False, ragged=False, masked=False, per_row=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["gated", "gated", "sandwich", "sandwich", "distil", "distil"])
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    params = rng.choice(["f32", kind])
    if call == "gated":
        case = dict(call=call, T=_log(rng, 1, 16384), K=_log(rng, 8, 8192), H=_log(rng, 8, 8192), type=kind, params=params,
                    bias=rng.random() < 0.5, act=rng.choice(ACTIVATIONS), grad=rng.random() < 0.6)
        if case["act"] == "relu" and case["grad"] and kind == "f32":
            # (which side of zero a sum near it is on decides over a whole term of a gradient, and 32 bits do not)
            case["act"] = "silu"
        if rng.random() < 0.5:
            case.update(K=(case["K"] + 15) // 16 * 16, H=(case["H"] + 15) // 16 * 16)
        rows = "T"
    elif call == "sandwich":
        case = dict(call=call, rows=_log(rng, 1, 131072), C=_log(rng, 10, 16384), type=kind, params=params,
                    gate=rng.choice(["none", "row", "all"]), grad=rng.random() < 0.7)
        if case["grad"]:
            # (which neighbour of 16 bits an element of the stream is rounded to shows in parameters' gradients of 32 bits)
            case["params"] = kind
        rows = "rows"
    else:
        case = dict(call=call, rows=_log(rng, 1, 32768), V=_log(rng, 10, 131072), k=_log(rng, 1, 128), type=kind,
                    tau=rng.choice([1.0, 1.0, 2.0, 4.0]), labels=rng.random() < 0.5, ragged=rng.random() < 0.5,
                    masked=rng.random() < 0.3, per_row=rng.random() < 0.5)
        case["k"] = min(case["k"], case["V"] // 2)
        rows = "rows"
    most = [work(c) for c in listed() if c["call"] == call]
    while case[rows] > 1 and any(work(case)[w] > max(m[w] for m in most) for w in ("bytes", "flops")):
        case[rows] = max(1, case[rows] // 2)
    return case


def work(case):
    size = SIZES[case["type"]]
    if case["call"] == "gated":
        T, K, H = case["T"], case["K"], case["H"]
        rows, weights, param = size * T * (K + H), 2 * size * H * K, 2 * H * SIZES[case["params"]] * bool(case["bias"])
        times = 2 if case["grad"] else 1  # (every operand has a gradient of its size)
        return dict(bytes=times * (rows + weights + param), flops=(12 if case["grad"] else 4) * T * H * K)
    if case["call"] == "sandwich":
        n, C = case["rows"] * case["C"], case["C"]
        gate = {"none": 0, "row": case["rows"], "all": n}[case["gate"]]
        times = 2 if case["grad"] else 1
        return dict(bytes=times * (size * (4 * n + gate) + 5 * C * SIZES[case["params"]]), flops=(60 if case["grad"] else 20) * n)
    n = case["rows"] * case["V"]
    teacher = case["rows"] * case["k"] * (size + 8) + 8 * case["rows"] * bool(case["labels"])
    return dict(bytes=2 * size * n + teacher + 4 * case["rows"], flops=(16 if case["labels"] and case["tau"] != 1.0 else 10) * n)


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _activations(rows, C, kind, f):
    x = torch.randn(rows, C, **f)
    return x.mul_(torch.rand(rows, 1, **f).mul_(2).add_(0.5)).add_(torch.randn(rows, 1, **f)).to(TYPES[kind])


def _prepare_gated(case, s, f):
    T, K, H, t, p = case["T"], case["K"], case["H"], TYPES[case["type"]], TYPES[case["params"]]
    s["x"] = torch.randn(T, K, **f).to(t)
    for name in ("gate", "up"):
        s["w_" + name] = (torch.randn(H, K, **f) / math.sqrt(K)).to(t)
        s["b_" + name] = (0.5 * torch.randn(H, **f)).to(p) if case["bias"] else None
    if case["grad"]:
        s["dy"] = torch.randn(T, H, **f).to(t)
    return ["x", "w_gate", "w_up", "b_gate", "b_up"]


def _prepare_sandwich(case, s, f):
    rows, C, t, p = case["rows"], case["C"], TYPES[case["type"]], TYPES[case["params"]]
    s["x"], s["residual"] = _activations(rows, C, case["type"], f), _activations(rows, C, case["type"], f)
    s["gate"] = None
    if case["gate"] != "none":
        s["gate"] = torch.sigmoid(torch.randn(rows, 1 if case["gate"] == "row" else C, **f)).to(t)
    s["scale"] = (0.5 + 0.1 * torch.randn(C, **f)).to(p)
    s["w1"], s["w2"] = [(1 + 0.1 * torch.randn(C, **f)).to(p) for _ in range(2)]
    s["b1"], s["b2"] = [(0.1 * torch.randn(C, **f)).to(p) for _ in range(2)]
    if case["grad"]:
        s["dy"], s["dh"] = [torch.randn(rows, C, **f).to(t) for _ in range(2)]
    return ["x", "residual", "gate", "scale", "w1", "b1", "w2", "b2"]


def _prepare_distil(case, s, f):
    rows, V, k, t = case["rows"], case["V"], case["k"], TYPES[case["type"]]
    student = 2 * torch.randn(rows, V, **f)
    teacher = 0.5 * student + 2 * torch.randn(rows, V, **f)
    if case["masked"]:
        gone = torch.rand(V, **f) < 0.1
        gone[:case["k"] + 1] = False
        student.masked_fill_(gone, -math.inf)
        teacher.masked_fill_(gone, -math.inf)
    values, indices = teacher.topk(k, dim=1)
    s["targets"] = None
    if case["labels"]:
        s["targets"] = indices[:, 0].clone()
    if case["ragged"]:
        length = torch.randint(0, k + 1, (rows, 1), **f)
        indices = torch.where(torch.arange(k, device="cuda") < length, indices, -1)
        if case["labels"]:
            s["targets"] = torch.where(torch.rand(rows, **f) < 0.1, -1, s["targets"])
    s["x"], s["values"], s["indices"] = student.to(t), values.to(t), indices
    # (a program whose gradients have 16 bits with a short exponent scales its loss)
    s["dy"] = torch.rand(rows, **f) if case["per_row"] else torch.full((), 4.0 * rows if case["type"] == "f16" else 1.0, device="cuda")
    if case["type"] == "f16" and case["per_row"]:
        s["dy"] *= 4.0
    return ["x"]


def prepare(case, seed):
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    s = dict(case=case, dtype=TYPES[case["type"]])
    wanted = {"gated": _prepare_gated, "sandwich": _prepare_sandwich, "distil": _prepare_distil}[case["call"]](case, s, f)
    s["wanted"] = [n for n in wanted if s[n] is not None and "dy" in s]
    for name in s["wanted"]:
        s[name] = s[name].detach().requires_grad_()
    return s


MIX = 0.3


# ---- the plain forms ----------------------------------------------------------------------------------------------------------
def _plain_activation(g, act):
    """(act(g), its derivative)"""
    if act == "relu":
        return torch.relu(g), (g > 0).float()
    if act == "gelu":
        half = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * half, half + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def _plain_gated(s, c, t):
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if c["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    a, da = _plain_activation(g, c["act"])
    out = dict(y=(a * u).to(t))
    if c["grad"]:
        dy = s["dy"].float()
        dg, du = dy * u * da, dy * a
        out.update(dx=(dg @ wg + du @ wu).to(t), dw_gate=(dg.t() @ x).to(t), dw_up=(du.t() @ x).to(t))
        if c["bias"]:
            out.update(db_gate=dg.sum(0).to(s["b_gate"].dtype), db_up=du.sum(0).to(s["b_up"].dtype))
    return out


def _plain_normed(x):
    d = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * rstd, rstd


def _plain_norm_grad(a, z, rstd):
    return rstd * (a - a.mean(1, keepdim=True) - z * (a * z).mean(1, keepdim=True))


def _plain_sandwich(s, c, t):
    scale, w1, b1, w2, b2 = [s[n].float() for n in ("scale", "w1", "b1", "w2", "b2")]
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    z1, rstd1 = _plain_normed(s["x"].float())
    n1 = z1 * w1 + b1
    # the residual stream is held in its type, and that is what is normalised
    h = (s["residual"].float() + gate * scale * n1).to(t)
    z2, rstd2 = _plain_normed(h.float())
    out = dict(y=(z2 * w2 + b2).to(t), h=h)
    if c["grad"]:
        p, dy = s["w1"].dtype, s["dy"].float()
        dh = s["dh"].float() + _plain_norm_grad(dy * w2, z2, rstd2)
        dn1 = dh * gate * scale
        out.update(dx=_plain_norm_grad(dn1 * w1, z1, rstd1).to(t), dresidual=dh.to(t), dscale=(dh * gate * n1).sum(0).to(p),
                   dw1=(dn1 * z1).sum(0).to(p), db1=dn1.sum(0).to(p), dw2=(dy * z2).sum(0).to(p), db2=dy.sum(0).to(p))
        if s["gate"] is not None:
            dgate = dh * scale * n1
            out.update(dgate=(dgate.sum(1, keepdim=True) if c["gate"] == "row" else dgate).to(t))
    return out


def _plain_softmax(x):
    """(exp(x - largest) / sum, log of the sum of exp(x)) of rows with a number in them."""
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    return e / total, torch.log(total) + m


def _plain_distil(s, c, t):
    x, tau, rows = s["x"].float(), c["tau"], c["rows"]
    there = s["indices"] >= 0
    at = s["indices"].clamp_min(0)
    some = there.any(1, keepdim=True)
    part = 1 - MIX if c["labels"] else 1.0
    values = torch.where(there, s["values"].float() / tau, torch.where(some, -math.inf, 0.0))
    p, p_log = _plain_softmax(values)
    q, q_log = _plain_softmax(x / tau)
    terms = p * ((values - p_log) - (torch.gather(x, 1, at) / tau - q_log))
    loss = part * tau * tau * torch.where(there, terms, 0.0).sum(1)
    dy = s["dy"] if c["per_row"] else s["dy"] / rows
    weight = part * tau * some.float() * dy.view(-1, 1)
    dx = q * weight
    dx.scatter_add_(1, at, torch.where(there, -p * weight, 0.0))
    if c["labels"]:
        labelled = (s["targets"] >= 0).view(-1, 1)
        target = s["targets"].clamp_min(0).view(-1, 1)
        q, q_log = _plain_softmax(x)
        loss = loss + torch.where(labelled, MIX * (q_log - torch.gather(x, 1, target)), 0.0).view(-1)
        weight = MIX * labelled.float() * dy.view(-1, 1)
        dx.addcmul_(q, weight)
        dx.scatter_add_(1, target, -weight)
    return dict(loss=loss if c["per_row"] else loss.sum() / rows, dx=dx.to(t))


_PLAIN = {"gated": _plain_gated, "sandwich": _plain_sandwich, "distil": _plain_distil}


# ---- the framework's operators ----------------------------------------------------------------------------------------------------
def _framework(s):
    import l_inf_dist_net_v2_b200 as ldn
    c = s["case"]
    if c["call"] == "gated":
        out = dict(y=ldn.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=c["act"]))
        upstream = [s["dy"]] if c["grad"] else []
    elif c["call"] == "sandwich":
        y, h = ldn.sandwich_norm(s["x"], s["residual"], s["w2"], s["b2"], post_weight=s["w1"], post_bias=s["b1"], scale=s["scale"],
                                 gate=s["gate"], eps=EPS)
        out = dict(y=y, h=h)
        upstream = [s["dy"], s["dh"]] if c["grad"] else []
    else:
        out = dict(loss=ldn.distillation_loss(s["x"], s["values"], s["indices"], s["targets"], temperature=c["tau"],
                                              mix=MIX if c["labels"] else 0.0, reduction="none" if c["per_row"] else "mean"))
        upstream = [s["dy"]]
    if not upstream:
        return out
    grads = torch.autograd.grad(list(out.values()), [s[n] for n in s["wanted"]], upstream)
    return {**{n: v.detach() for n, v in out.items()}, **{"d" + n: g for n, g in zip(s["wanted"], grads)}}


def run(state):
    if own:
        return _framework(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["call"]](state, state["case"], state["dtype"])


# ---- 64 bits --------------------------------------------------------------------------------------------------------------------
def _exact_gated(c, d):
    project = lambda n: torch.einsum("tk,hk->th", d["x"], d["w_" + n]) + (d["b_" + n] if c["bias"] else 0.0)  # noqa: E731
    g, u = project("gate"), project("up")
    # each activation as g^m times a distribution's function, with its density: logistic, normal, a step at zero
    power = 0 if c["act"] == "sigmoid" else 1
    if c["act"] == "relu":
        cdf, pdf = (g > 0).double(), torch.zeros_like(g)
    elif c["act"] == "gelu":
        cdf, pdf = torch.special.ndtr(g), torch.exp(-g.square() / 2) / math.sqrt(math.tau)
    else:
        cdf = 1 / (1 + torch.exp(-g))
        pdf = cdf * torch.exp(-g) / (1 + torch.exp(-g))
    a = g ** power * cdf
    out = dict(y=a * u)
    if "dy" in d:
        du = d["dy"] * a
        dg = d["dy"] * u * (g ** power * pdf + power * cdf)
        out.update(dx=torch.einsum("th,hk->tk", dg, d["w_gate"]) + torch.einsum("th,hk->tk", du, d["w_up"]),
                   dw_gate=torch.einsum("th,tk->hk", dg, d["x"]), dw_up=torch.einsum("th,tk->hk", du, d["x"]))
        if c["bias"]:
            out.update(db_gate=dg.sum(0), db_up=du.sum(0))
    return out


def _exact_norm(x):
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sigma = (var + EPS).sqrt()
    return (x - mean) / sigma, sigma


def _exact_project(a, z, sigma):
    """`a` off the constant and off the normalised row"""
    a = a / sigma
    return a - a.mean(1, keepdim=True) - z * ((a * z).sum(1, keepdim=True) / z.size(1))


def _exact_sandwich(c, d, dtype):
    z1, sigma1 = _exact_norm(d["x"])
    weigh = d["scale"] * (d["gate"] if "gate" in d else 1.0)
    whole = d["residual"] + weigh * (z1 * d["w1"] + d["b1"])
    z2, sigma2 = _exact_norm(whole.to(dtype).double())
    out = dict(y=z2 * d["w2"] + d["b2"], h=whole)
    if "dy" in d:
        dh = d["dh"] + _exact_project(d["dy"] * d["w2"], z2, sigma2)
        branch = d["w1"] * z1 + d["b1"]
        out.update(dx=_exact_project(dh * weigh * d["w1"], z1, sigma1), dresidual=dh, dw1=torch.einsum("rc,rc->c", dh * weigh, z1),
                   db1=(dh * weigh).sum(0), dw2=torch.einsum("rc,rc->c", d["dy"], z2), db2=d["dy"].sum(0),
                   dscale=(dh * (d["gate"] if "gate" in d else 1.0) * branch).sum(0))
        if "gate" in d:
            dgate = dh * d["scale"] * branch
            out.update(dgate=dgate if c["gate"] == "all" else dgate.sum(1, keepdim=True))
    return out


def _exact_distil(c, d, s):
    x, tau, rows = d["x"], c["tau"], c["rows"]
    part = 1 - MIX if c["labels"] else 1.0
    # the teacher's distribution over the classes, a column behind them for what is not there
    at = torch.where(s["indices"] < 0, c["V"], s["indices"])
    some = (s["indices"] >= 0).any(1)
    logits = torch.full((rows, c["V"] + 1), -math.inf, device="cuda", dtype=torch.float64).scatter_(1, at, d["values"] / tau)[:, :-1]
    p = torch.nan_to_num(torch.softmax(logits, 1), nan=0.0)
    log_q = torch.log_softmax(x / tau, 1)
    loss = part * tau ** 2 * (torch.xlogy(p, p) - torch.where(p > 0, p * log_q, 0.0)).sum(1)
    dx = part * tau * (log_q.exp() * some.unsqueeze(1) - p)
    if c["labels"]:
        log_q, labelled = torch.log_softmax(x, 1), s["targets"] >= 0
        target = s["targets"].clamp_min(0).unsqueeze(1)
        loss = loss - MIX * torch.where(labelled, torch.gather(log_q, 1, target).squeeze(1), 0.0)
        dx += MIX * labelled.unsqueeze(1) * log_q.exp().scatter_add_(1, target, torch.full_like(target, -1.0, dtype=torch.float64))
    dx *= (d["dy"] if c["per_row"] else d["dy"].expand(rows) / rows).unsqueeze(1)
    return dict(loss=loss if c["per_row"] else loss.mean(), dx=dx)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if case["call"] == "gated":
        return _exact_gated(case, d)
    if case["call"] == "sandwich":
        return _exact_sandwich(case, d, s["dtype"])
    return _exact_distil(case, d, s)
