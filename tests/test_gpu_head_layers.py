"""The head's layers and models in the ways that a program uses them: differentiated again, recomputed, in mixed precision, moved,
answering in integers while their weights change, from several threads."""
import copy
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import l_inf_dist_net_v2_b200 as ldn
from l_inf_dist_net_v2_b200.optim import FusedAdam, FusedSGD

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _model(**kwargs):
    torch.manual_seed(0)
    model = ldn.ResidualModel(4, 96, [1, 8, 8], hidden=120, blocks=3, seed=11, **kwargs).cuda()
    ldn.set_p_norm(model, float("inf"))
    return model


def _images(n=40, seed=1):
    return torch.rand(n, 1, 8, 8, **_gen(seed))


# ---- differentiated again ---------------------------------------------------------------------------------------------------------
def _norm_case():
    f = _gen(1)
    x, r = (torch.randn(6, 40, **f).requires_grad_() for _ in range(2))
    w, b = (torch.randn(40, **f).requires_grad_() for _ in range(2))
    return x, r, w, b


def _again(tensor):
    with pytest.raises(RuntimeError, match="differentiated again"):
        tensor.square().sum().backward()


def test_a_norm_differentiated_twice_says_so():
    x, _, w, b = _norm_case()
    v = torch.randn(6, 40, **_gen(2))
    plain = torch.autograd.grad((ldn.layer_norm(x, w, b) * v).sum(), (x, w, b))
    for weight in (w, w.detach(), None):
        y = ldn.layer_norm(x, weight, b)
        gx, = torch.autograd.grad((y * v).sum(), x, create_graph=True)
        assert gx.requires_grad
        _again(gx)
    gx, gw, gb = torch.autograd.grad((ldn.layer_norm(x, w, b) * v).sum(), (x, w, b), create_graph=True)
    assert all(torch.equal(s, t) for s, t in zip((gx, gw, gb), plain))
    _again(gw)
    # through what is in front of the norm
    z = ldn.layer_norm(x * 2, w, b)
    gx, = torch.autograd.grad(z.sum(), x, create_graph=True)
    _again(gx)
    # a gradient that depends on nothing that is differentiated is one
    gw, = torch.autograd.grad((ldn.layer_norm(x.detach(), w, b) * v).sum(), w, create_graph=True)
    assert not gw.requires_grad and torch.equal(gw, plain[1])


def test_the_joined_norm_differentiated_twice_says_so():
    x, r, w, b = _norm_case()
    v = torch.randn(6, 40, **_gen(2))
    for leaves, wanted in [((x, r, w, b), x), ((x, r, w, b), r), ((x, r, w, b), w), ((x.detach(), r, w.detach(), b), r)]:
        y, h = ldn.dropout_add_layer_norm(*leaves, 0.3, 5)
        plain, = torch.autograd.grad((y * v).sum(), wanted, retain_graph=True)
        g, = torch.autograd.grad((y * v).sum(), wanted, create_graph=True)
        assert torch.equal(g, plain)
        _again(g)
    y, _ = ldn.dropout_add_layer_norm(x.detach(), r.detach(), w, b, 0.3, 5)
    gw, = torch.autograd.grad((y * v).sum(), w, create_graph=True)
    assert not gw.requires_grad


# ---- recomputed ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_head_has_the_gradients_of_its_masks(reentrant):
    a = _model(dropout=0.4).head
    b = copy.deepcopy(a)
    xs = [torch.randn(30, 96, **_gen(k)).requires_grad_() for k in range(2)]
    outs, wants = [checkpoint(a, x, use_reentrant=reentrant) for x in xs], [b(x) for x in xs]
    for out, want, x in zip(outs, wants, xs):
        assert torch.equal(out, want)
        out.square().sum().backward()
        g, x.grad = x.grad, None
        want.square().sum().backward()
        assert torch.equal(x.grad, g)
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(a.parameters(), b.parameters()))


# ---- mixed precision -----------------------------------------------------------------------------------------------------------------
# seven products whose operands and results are rounded to eight bits (2^-9 each), and as many times the stream and the norms in 16
# bits: of the largest logit
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_model_under_autocast(dtype):
    model, x = _model(dropout=0.2), _images()
    plain = copy.deepcopy(model)
    want = plain(x)
    with torch.autocast("cuda", dtype=dtype):
        got = model(x)
        loss = torch.nn.functional.cross_entropy(got, torch.arange(40, device="cuda") % 10)
    assert got.dtype == dtype and (got - want).abs().max() <= 7 * 3 * 2.0 ** -9 * want.abs().max()
    loss.backward()
    assert all(p.grad is not None and p.grad.dtype == F32 and p.grad.isfinite().all() for p in model.head.parameters())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_head_in_16_bits_behind_distance_layers(dtype):
    model, x = _model(dropout=0.2), _images()
    want = copy.deepcopy(model)(x)
    model.head.to(dtype)
    got = model(x)
    assert got.dtype == dtype and (got - want).abs().max() <= 7 * 6 * 2.0 ** -9 * want.abs().max()
    torch.nn.functional.cross_entropy(got.float(), torch.arange(40, device="cuda") % 10).backward()
    assert all(p.grad is not None and p.grad.dtype == dtype and p.grad.isfinite().all() for p in model.head.parameters())
    whole = copy.deepcopy(model).eval()  # (with the running means of the step above)
    whole.head.float()
    with torch.no_grad():
        want = whole(x)
    answer = model.quantize()(x)
    assert (answer - want).abs().max() <= 0.1 * want.abs().max()


# ---- answering -------------------------------------------------------------------------------------------------------------------------
def _fresh(model, x):
    """What the model's weights of now answer in integers."""
    with torch.no_grad():
        features, _, _ = model.fc_dist((x.flatten(1), None, None))
        return model.head.quantized()(features)


def test_integers_last_until_train():
    model, x = _model(), _images()
    want = _fresh(model.eval(), x)
    model.quantize()
    for answers in (model, model.eval(), model.train(False), copy.deepcopy(model)):
        with torch.no_grad():
            assert torch.equal(answers(x), want)
        y = answers(x)  # integers without torch.no_grad(), too, and no gradient
        assert torch.equal(y, want) and not y.requires_grad
    model.train()
    assert model(x).requires_grad
    with torch.no_grad():
        assert not torch.equal(model.eval()(x), want)


@pytest.mark.parametrize("change", ["load", "adam", "sgd", "torch", "copy", "part", "to", "half and back"])
def test_integers_are_those_of_the_weights(change):
    model, x = _model(), _images()
    torch.nn.functional.cross_entropy(model(x), torch.arange(40, device="cuda") % 10).backward()
    before = model.quantize()(x)
    if change == "load":
        torch.manual_seed(5)
        model.load_state_dict(ldn.ResidualModel(4, 96, [1, 8, 8], hidden=120, blocks=3).cuda().state_dict())
    elif change in ("adam", "sgd", "torch"):
        make = dict(adam=FusedAdam, sgd=FusedSGD, torch=torch.optim.SGD)[change]
        make(model.head.parameters(), lr=0.05).step()
    elif change == "copy":
        with torch.no_grad():
            model.head.final.weight.mul_(2)
    elif change == "part":
        model.head.up[1] = torch.nn.Linear(96, 120, device="cuda")
    elif change == "to":
        model.cpu()
        model.cuda()
    else:
        model.head.half().float()
    after = model(x)
    assert torch.equal(after, _fresh(model, x)) and torch.equal(after, before) == (change == "to")


# ---- an integer layer that is moved -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("terms", [96, 100])
def test_an_integer_layer_that_is_moved(terms):
    layer = ldn.Int8Linear(torch.randn(30, terms, **_gen(1)), torch.randn(30, **_gen(2)), "relu")
    x = torch.randn(9, terms, **_gen(3))
    want = layer(x)
    for moved in (copy.deepcopy(layer), copy.deepcopy(layer).cpu().cuda(), copy.deepcopy(layer).half(), copy.deepcopy(layer).cpu().bfloat16().cuda(),
                  torch.nn.Sequential(copy.deepcopy(layer)).cpu().cuda()[0]):
        assert moved.weight.stride() == layer.weight.stride() and moved.weight_scale.dtype == moved.bias.dtype == F32
        assert torch.equal(moved(x), want) and moved.state_dict().keys() == layer.state_dict().keys()


@pytest.mark.parametrize("move", [lambda m: m.half(), lambda m: m.cpu().cuda(), lambda m: m.to(torch.bfloat16), lambda m: m.double()])
def test_an_integer_head_that_is_moved(move):
    head = _model().head.quantized()
    h = torch.randn(20, 96, **_gen(1))
    want = head(h)
    moved = move(copy.deepcopy(head))
    assert torch.equal(moved(h), want) and moved(h.half()).dtype == F16
    assert all(b.dtype in (F32, torch.int8) for b in moved.buffers())


# ---- threads ---------------------------------------------------------------------------------------------------------------------------------
def test_several_threads():
    weight = ldn.quantize_rows(torch.randn(130, 500, **_gen(1)))

    def work(k):
        x, r = (torch.randn(40 + 90 * k, 500, **_gen(10 * k + i)).requires_grad_() for i in (2, 3))
        w, b = (torch.randn(500, **_gen(10 * k + i)).requires_grad_() for i in (4, 5))
        y, h = ldn.dropout_add_layer_norm(x, r, w, b, 0.2, k)
        d = ldn.dropout(ldn.layer_norm(h, w, b), 0.1, k, 1)
        grads = torch.autograd.grad((y, d), (x, r, w, b), (x.detach(), r.detach()))
        with torch.no_grad():
            return (y, h, d) + grads + (ldn.int8_linear(x, weight), ldn.int8_linear(ldn.layer_norm_quantized(x, w, b), weight))
    wants = [work(k) for k in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def repeat(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(25):
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
