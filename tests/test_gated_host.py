"""The gated head's layers with torch operations in place of the kernels, and what its operators refuse without a GPU."""
import copy
import ctypes
import math
import os
import re

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import l_inf_dist_net_v2_b200 as ldn
from head_stand_in import RowOperators
from l_inf_dist_net_v2_b200 import head as head_module
from l_inf_dist_net_v2_b200 import losses
from l_inf_dist_net_v2_b200._lib import lib
from l_inf_dist_net_v2_b200.parallel import OverlappedDataParallel

BAD = 1


@pytest.fixture
def on_the_host(monkeypatch):
    monkeypatch.setattr(head_module, "_native", lambda: RowOperators)


def _head(**kwargs):
    torch.manual_seed(0)
    return ldn.GatedHead(12, 20, num_classes=5, blocks=2, seed=7, **{"dropout": 0.25, **kwargs})


def test_the_data_parallel_wrapper_updates_every_layer(on_the_host):
    a = _head(dropout=0.0)
    b = copy.deepcopy(a)
    make = lambda params: torch.optim.Adam(params, lr=0.02)  # noqa: E731
    wrapper, plain = OverlappedDataParallel(a, make), make(list(b.parameters()))
    start = [p.detach().clone() for p in a.parameters()]
    gen = torch.Generator().manual_seed(0)
    for _ in range(4):
        x, t = torch.randn(8, 12, generator=gen), torch.randint(0, 5, (8,), generator=gen)
        logits = a(x)
        torch.nn.functional.cross_entropy(logits, t).backward()
        wrapper.step()
        plain.zero_grad(set_to_none=True)
        want = b(x)
        torch.nn.functional.cross_entropy(want, t).backward()
        plain.step()
        assert torch.allclose(logits, want, rtol=0, atol=1e-6)
    wrapper.finish()
    for p, q, s in zip(a.parameters(), b.parameters(), start):
        assert torch.allclose(p, q, rtol=0, atol=1e-6) and not torch.equal(p, s)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_head_has_the_gradients_of_its_masks(on_the_host, reentrant):
    a = _head()
    b = copy.deepcopy(a)
    x = torch.randn(30, 12).requires_grad_()
    out, want = checkpoint(a, x, use_reentrant=reentrant), b(x)
    assert torch.equal(out, want)
    g, = torch.autograd.grad(out.square().sum(), x) if not reentrant else (None,)
    if reentrant:
        out.square().sum().backward()
        g, x.grad = x.grad, None
    assert torch.equal(g, torch.autograd.grad(want.square().sum(), x)[0])


def test_the_head_keeps_its_state_and_its_type(on_the_host):
    a, b = _head(activation="gelu"), _head(activation="gelu")
    with torch.no_grad():
        for p in a.parameters():
            p.add_(0.1)
    b.load_state_dict(a.state_dict())
    x = torch.randn(6, 12)
    with torch.no_grad():
        assert torch.equal(a.eval()(x), b.eval()(x)) and a.eval()(x).dtype == torch.float32
        assert a.bfloat16()(x).dtype == torch.bfloat16


def test_a_gated_model_has_no_integers():
    model = ldn.ResidualModel(3, 16, [1, 2, 2], hidden=8, blocks=1, gated=True)
    assert isinstance(model.head, ldn.GatedHead) and model.training
    with pytest.raises(RuntimeError, match="floating point"):
        model.quantize()
    assert model.training and not model._integers


def test_values_that_make_no_sense_are_refused():
    x, w, i = torch.rand(4, 8), torch.rand(3, 8), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="activation"):
        ldn.gated_linear(x, w, w, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        ldn.GatedLinear(8, 3, "none")
    with pytest.raises(ValueError, match="reduction"):
        ldn.distillation_loss(x, x[:, :2], i, reduction="average")
    with pytest.raises(ValueError, match="targets"):
        ldn.distillation_loss(x, x[:, :2], i, mix=0.5)
    for call in (lambda: ldn.gated_linear(x, w, w), lambda: ldn.sandwich_norm(x, x), lambda: ldn.distillation_loss(x, x[:, :2], i),
                 lambda: losses.distillation()(x, (x[:, :2], i), i[:, 0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


HERE = ctypes.create_string_buffer(256)
AT = ctypes.c_void_p((ctypes.addressof(HERE) + 31) // 32 * 32)
# (whatever stands where a pointer is wanted: none of these calls may launch anything)
LONG = 2 ** 31 - 1


@pytest.mark.parametrize("change", [dict(K=0), dict(H=0), dict(rows=-1), dict(type=3), dict(activation=0), dict(activation=2), dict(activation=6),
                                    dict(param_type=1), dict(x=None), dict(w_gate=None), dict(w_up=None), dict(y=None), dict(u=None),
                                    dict(pitch_gate=3), dict(pitch_up=3), dict(pitch_saved=15), dict(pitch_saved=24), dict(rows=LONG),
                                    dict(K=LONG), dict(H=LONG), dict(g=ctypes.c_void_p(AT.value + 4))])
def test_gated_arguments(change):
    a = dict(x=AT, pitch=4, rows=2, K=4, H=20, type=0, w_gate=AT, pitch_gate=4, w_up=AT, pitch_up=4, b_gate=AT, b_up=None, param_type=0,
             activation=3, y=AT, g=AT, u=AT, pitch_saved=32, images=None, stream=None)
    assert lib.ldn_gated_linear(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(K=0), dict(type=-1), dict(activation=2), dict(grad_y=None), dict(g=None), dict(u=None), dict(x=None),
                                    dict(w_gate=None), dict(grad_w_up=None), dict(pitch_saved=20), dict(param_type=2)])
def test_gated_backward_arguments(change):
    a = dict(grad_y=AT, x=AT, pitch=4, rows=2, K=4, H=20, type=0, w_gate=AT, pitch_gate=4, w_up=AT, pitch_up=4, g=AT, u=AT, pitch_saved=32, images=None,
             activation=3, grad_x=AT, grad_w_gate=AT, grad_w_up=AT, grad_b_gate=AT, grad_b_up=AT, param_type=0, stream=None)
    assert lib.ldn_gated_linear_backward(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(C=0), dict(C=LONG), dict(rows=-1), dict(type=3), dict(param_type=1), dict(eps=-1.0), dict(eps=math.nan),
                                    dict(gate_kind=3), dict(gate_kind=-1), dict(gate=None), dict(x=None), dict(residual=None), dict(h=None),
                                    dict(y=None)])
def test_sandwich_arguments(change):
    a = dict(x=AT, pitch=4, residual=AT, pitch_residual=4, gate=AT, pitch_gate=1, gate_kind=1, rows=2, C=4, type=0, scale=None, post_weight=AT,
             post_bias=AT, weight=AT, bias=AT, param_type=0, eps=1e-5, h=AT, y=AT, stats=None, stream=None)
    assert lib.ldn_sandwich_norm(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(C=0), dict(type=3), dict(param_type=2), dict(gate_kind=5), dict(gate=None), dict(x=None), dict(h=None),
                                    dict(stats=None), dict(grad_y=None, grad_h=None)])
def test_sandwich_backward_arguments(change):
    a = dict(grad_y=AT, grad_h=AT, x=AT, pitch=4, h=AT, gate=AT, pitch_gate=1, gate_kind=1, rows=2, C=4, type=0, scale=None, post_weight=AT,
             post_bias=AT, weight=AT, param_type=0, stats=AT, grad_x=AT, grad_residual=AT, grad_gate=AT, grad_scale=None, grad_post_weight=AT,
             grad_post_bias=AT, grad_weight=AT, grad_bias=AT, stream=None)
    assert lib.ldn_sandwich_norm_backward(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(V=0), dict(V=LONG), dict(rows=-1), dict(rows=LONG), dict(type=3), dict(value_type=-1), dict(k=0),
                                    dict(k=1025), dict(tau=0.0), dict(tau=-1.0), dict(tau=math.inf), dict(tau=math.nan), dict(x=None),
                                    dict(values=None), dict(indices=None), dict(losses=None)])
def test_distillation_arguments(change):
    a = dict(x=AT, pitch=4, rows=2, V=4, type=0, values=AT, value_type=0, indices=AT, k=2, targets=None, tau=1.0, part=1.0, mix=0.0, losses=AT,
             stats=None, loss_scale=1.0, loss=None, stream=None)
    assert lib.ldn_distillation(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(V=0), dict(k=0), dict(tau=0.0), dict(x=None), dict(stats=None), dict(up=None), dict(grad=None)])
def test_distillation_backward_arguments(change):
    a = dict(x=AT, pitch=4, rows=2, V=4, type=0, values=AT, value_type=0, indices=AT, k=2, targets=None, tau=1.0, part=1.0, mix=0.0, stats=AT,
             up=AT, up_per_row=0, up_scale=1.0, grad=AT, stream=None)
    assert lib.ldn_distillation_backward(*{**a, **change}.values()) == BAD


def test_calls_without_rows_do_nothing():
    assert lib.ldn_gated_linear(None, 4, 0, 4, 4, 0, None, 4, None, 4, None, None, 0, 3, None, None, None, 0, None, None) == 0
    assert lib.ldn_sandwich_norm(None, 4, None, 4, None, 0, 0, 0, 4, 0, None, None, None, None, None, 0, 1e-5, None, None, None, None) == 0
    assert lib.ldn_distillation_backward(None, 4, 0, 4, 0, None, 0, None, 2, None, 1.0, 1.0, 0.0, None, None, 0, 1.0, None, None) == 0


def test_the_kinds_of_gates_are_what_the_header_says():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "ldn_b200.h")) as f:
        header = f.read()
    kinds = dict(re.findall(r"#define (LDN_GATE_\w+) (\d+)", header))
    assert kinds == dict(LDN_GATE_NONE="0", LDN_GATE_ROW="1", LDN_GATE_ALL="2")
    for name, number in re.findall(r"(LDN_GATE_\w+) \((\d+)\)", header):  # (as comments number them)
        assert kinds[name] == number
