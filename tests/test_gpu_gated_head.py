"""The gated head and its distillation as a program uses them: whole steps, in mixed precision, recorded, recomputed, from several threads."""
import copy
import os
import re
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import l_inf_dist_net_v2_b200 as ldn
from head_oracle import EPS32
from l_inf_dist_net_v2_b200 import losses
from l_inf_dist_net_v2_b200.optim import FusedAdam

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _model(**kwargs):
    torch.manual_seed(0)
    model = ldn.ResidualModel(4, 96, [1, 8, 8], hidden=120, blocks=3, seed=11, gated=True, **{"dropout": 0.0, **kwargs}).cuda()
    ldn.set_p_norm(model, float("inf"))
    return model


def _images(n=40, seed=1):
    return torch.rand(n, 1, 8, 8, **_gen(seed))


def _teacher(n=40, classes=10, k=4, seed=2):
    return tuple(torch.randn(n, classes, **_gen(seed)).mul(2).topk(k))


def _plain_head(head, h):
    """In 64 bits, without dropout."""
    lin = lambda m, v: v @ m.weight.double().t() + m.bias.double()  # noqa: E731
    norm = lambda v, w, b: torch.nn.functional.layer_norm(v, v.shape[-1:], w.double(), b.double(), 1e-5)  # noqa: E731
    h = h.double()
    y = norm(h, head.norm.weight, head.norm.bias)
    for wide, down, gate, join in zip(head.wide, head.down, head.gate, head.join):
        g = y @ wide.weight_gate.double().t() + wide.bias_gate.double()
        f = lin(down, torch.nn.functional.silu(g) * (y @ wide.weight_up.double().t() + wide.bias_up.double()))
        h = h + torch.sigmoid(lin(gate, y)) * join.scale.double() * norm(f, join.post_weight, join.post_bias)
        y = norm(h, join.weight, join.bias)
    return lin(head.final, y)


def _plain_loss(logits, teacher, targets, tau, mix):
    q = torch.log_softmax(logits / tau, 1)
    p = torch.softmax(teacher[0].double() / tau, 1)
    kl = (p * (p.log() - q.gather(1, teacher[1]))).sum(1).mean()
    return (1 - mix) * tau ** 2 * kl + mix * torch.nn.functional.cross_entropy(logits, targets)


def test_a_head_and_its_loss_are_their_formulas():
    head, features = _model().head, torch.randn(50, 96, **_gen(1)).requires_grad_()
    with torch.no_grad():
        for join in head.join:
            join.scale.uniform_(0.2, 1.0)
    teacher, targets = _teacher(50), torch.arange(50, device="cuda") % 10
    got = head(features)
    want = _plain_head(head, features)
    # four products of up to 120 terms, three blocks: some hundred roundings of numbers of the stream's size
    assert (got - want).abs().max() <= 1000 * EPS32 * want.abs().max()
    loss = losses.distillation(4.0, 0.1)(got, teacher, targets)
    exact = _plain_loss(want, teacher, targets, 4.0, 0.1)
    # (the logits' errors, tau times as they are)
    assert abs(loss - exact) <= 4000 * EPS32 * (want.abs().max() + exact.abs())
    params = list(head.parameters())
    for a, b in zip(torch.autograd.grad(loss, [features] + params), torch.autograd.grad(exact, [features] + params)):
        assert (a - b).abs().max() <= 8000 * EPS32 * b.abs().max().clamp_min(1e-6)


def test_a_model_trains_and_answers():
    model, x, teacher, targets = _model(dropout=0.2), _images(), _teacher(), torch.arange(40, device="cuda") % 10
    optimizer = FusedAdam(model.parameters(), lr=1e-3)
    criterion = losses.distillation(4.0, 0.1)
    before = [p.detach().clone() for p in model.parameters()]
    for _ in range(5):
        loss = criterion(model(x), teacher, targets)
        optimizer.zero_grad()
        loss.backward()
        assert loss.isfinite() and all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
        optimizer.step()
    assert all(not torch.equal(p, b) for p, b in zip(model.head.parameters(), before[-len(list(model.head.parameters())):]))
    with torch.no_grad():
        want = model.eval()(x)
        again = _model()
        again.load_state_dict(model.state_dict())
        assert torch.equal(again.eval()(x), want) and torch.equal(model(x), want)
        # one image: another kernel for the projections
        assert (model(x[:1]) - want[:1]).abs().max() <= 1000 * EPS32 * want.abs().max()


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_head_has_the_gradients_of_its_masks(reentrant):
    a = _model(dropout=0.4).head
    b = copy.deepcopy(a)
    x = torch.randn(30, 96, **_gen(3)).requires_grad_()
    out, want = checkpoint(a, x, use_reentrant=reentrant), b(x)
    assert torch.equal(out, want)
    out.square().sum().backward()
    g, x.grad = x.grad, None
    want.square().sum().backward()
    assert torch.equal(x.grad, g) and all(torch.equal(p.grad, q.grad) for p, q in zip(a.parameters(), b.parameters()))


# (four products whose operands and results are rounded to eight bits, 2^-9 each, and as many times the stream and the norms in 16 bits, of the
# largest logit)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_model_under_autocast_and_in_16_bits(dtype):
    model, x = _model(), _images()
    want = copy.deepcopy(model)(x)
    auto = copy.deepcopy(model)
    with torch.autocast("cuda", dtype=dtype):
        got = auto(x)
        loss = losses.distillation()(got, _teacher(), torch.arange(40, device="cuda") % 10)
    assert got.dtype == dtype and (got - want).abs().max() <= 13 * 3 * 2.0 ** -9 * want.abs().max()
    loss.backward()
    assert all(p.grad is not None and p.grad.dtype == F32 and p.grad.isfinite().all() for p in auto.head.parameters())
    model.head.to(dtype)
    got = model(x)
    assert got.dtype == dtype and (got - want).abs().max() <= 13 * 6 * 2.0 ** -9 * want.abs().max()
    losses.distillation()(got, _teacher(), torch.arange(40, device="cuda") % 10).backward()
    assert all(p.grad is not None and p.grad.dtype == dtype and p.grad.isfinite().all() for p in model.head.parameters())


# ---- streams, graphs, threads ---------------------------------------------------------------------------------------------------------
def _leaves(dtype, seed=1, T=70, K=200, H=136, V=300):
    f = _gen(seed)
    shapes = [(T, K), (H, K), (H, K), (H,), (H,), (K, H), (T, K), (T, 1), (K,), (K,), (K,), (V, K)]
    return [(torch.randn(*s, **f) / s[-1] ** 0.5 if i not in (0, 6) else torch.randn(*s, **f)).to(dtype).requires_grad_() for i, s in enumerate(shapes)]


def _step(leaves, teacher, targets):
    """Everything in one pass, forward and backward."""
    x, wg, wu, bg, bu, wd, r, gate, scale, w1, w2, wf = leaves
    f = torch.nn.functional.linear(ldn.gated_linear(x, wg, wu, bg, bu), wd)
    y, h = ldn.sandwich_norm(f, r, w2, None, w1, None, scale, gate)
    loss = ldn.distillation_loss(torch.nn.functional.linear(y, wf), *teacher, targets, 2.0, 0.3) + 0.01 * h.float().square().mean()
    return (loss.detach(),) + torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recorded_in_graphs(dtype):
    """Two recorded steps of the same leaves on one stream, whose scratch they share, replayed in turn and between eager steps."""
    leaves, teacher, targets = _leaves(dtype), _teacher(70, 300), torch.arange(70, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = _step(leaves, teacher, targets)
    torch.cuda.synchronize()
    del want
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph, stream=stream):
            got.append(_step(leaves, teacher, targets))
    for turn in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(70, 200, **_gen(20 + turn)).to(dtype))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        eager = _step(leaves, teacher, targets)
        for outputs in got:
            assert all(torch.equal(a, b) for a, b in zip(outputs, eager))


def test_another_stream_and_several_threads():
    work = lambda k: _step(_leaves(F32, seed=k, T=30 + 50 * k), _teacher(30 + 50 * k, 300, seed=k), torch.arange(30 + 50 * k, device="cuda"))  # noqa: E731
    wants = [work(k) for k in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def repeat(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    if not all(torch.equal(s, t) for s, t in zip(work(k), wants[k])):
                        wrong.append(k)
            stream.synchronize()
        except Exception as e:  # (a thread's own end says nothing to the test)
            wrong.append(e)
    threads = [threading.Thread(target=repeat, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_the_example_of_the_documentation():
    """The code of INTEGRATION.md's section on the gated head, as it is written, on what its names stand for."""
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")) as f:
        section = f.read().split("## 7. ")[1].split("\n## ")[0]
    code, = re.findall(r"```python\n(.*?)```", section, re.S)
    f = _gen(5)
    names = dict(torch=torch, ldn=ldn, x=torch.randn(12, 96, **f), residual=torch.randn(12, 96, **f), weight=torch.ones(96, device="cuda"),
                 bias=torch.zeros(96, device="cuda"), w1=torch.ones(96, device="cuda"), b1=torch.zeros(96, device="cuda"),
                 s=torch.full((96,), 0.1, device="cuda"), g=torch.rand(12, 1, **f), images=torch.rand(12, 3, 32, 32, **f))
    for name in ("gate", "up"):
        names["weight_" + name], names["bias_" + name] = torch.randn(40, 96, **f), torch.randn(40, **f)
    with torch.device("cuda"):
        names["teacher"] = torch.nn.Sequential(torch.nn.Flatten(), torch.nn.LazyLinear(10))
    with torch.no_grad():
        logits = names["teacher"](names["images"])
    names["logits"], (names["values"], names["indices"]), names["targets"] = logits, logits.topk(3), logits.argmax(1)
    with torch.device("cuda"):
        exec(code, names)
    assert names["y"].shape == names["h"].shape == (12, 96) and names["loss"].isfinite()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in names["model"].head.parameters())
