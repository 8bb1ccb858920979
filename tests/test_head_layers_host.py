"""The head's layers as a program uses them (data-parallel training, recomputation, ranks), with torch operations in place of the
kernels, and sizes that the library refuses."""
import copy
import ctypes
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch.utils.checkpoint import checkpoint

import l_inf_dist_net_v2_b200 as ldn
from head_stand_in import RowOperators
from l_inf_dist_net_v2_b200 import head as head_module
from l_inf_dist_net_v2_b200._lib import lib
from l_inf_dist_net_v2_b200.parallel import OverlappedDataParallel, allreduce_mean_

BAD = 1


@pytest.fixture
def on_the_host(monkeypatch):
    monkeypatch.setattr(head_module, "_native", lambda: RowOperators)


def _head(**kwargs):
    torch.manual_seed(0)
    return ldn.ResidualHead(12, 20, num_classes=5, blocks=2, seed=7, **{"dropout": 0.25, **kwargs})


# ---- the data-parallel wrapper ----------------------------------------------------------------------------------------------------
def _train_both_ways(rank):
    """Four steps: with the wrapper, whose updates wait for a layer's next forward, and in the plain order."""
    a = _head()
    b = copy.deepcopy(a)
    make = lambda params: torch.optim.Adam(params, lr=0.02)  # noqa: E731
    wrapper, plain = OverlappedDataParallel(a, make), make(list(b.parameters()))
    start = [p.detach().clone() for p in a.parameters()]
    gen = torch.Generator().manual_seed(rank)
    for _ in range(4):
        x, t = torch.randn(8, 12, generator=gen), torch.randint(0, 5, (8,), generator=gen)
        logits = a(x)
        torch.nn.functional.cross_entropy(logits, t).backward()
        wrapper.step()
        plain.zero_grad(set_to_none=True)
        want = b(x)
        torch.nn.functional.cross_entropy(want, t).backward()
        if dist.is_initialized():
            allreduce_mean_([p.grad for p in b.parameters()])
        plain.step()
        if not torch.allclose(logits, want, rtol=0, atol=1e-6):
            return False
    wrapper.finish()
    return all(torch.allclose(p, q, rtol=0, atol=1e-6) and not torch.equal(p, s) and p.grad is None
               for p, q, s in zip(a.parameters(), b.parameters(), start))


def test_the_data_parallel_wrapper_updates_every_layer(on_the_host):
    assert _train_both_ways(0)


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _ranks(rank, world, port, out_dir, what):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    head_module._native = lambda: RowOperators
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        with open(os.path.join(out_dir, str(rank)), "w") as f:
            f.write(str(what(rank)))
    finally:
        dist.destroy_process_group()


def _on_two_ranks(tmp_path, what):
    mp.spawn(_ranks, args=(2, _free_port(), str(tmp_path), what), nprocs=2, join=True)
    return [(tmp_path / str(r)).read_text() for r in range(2)]


def test_the_data_parallel_wrapper_updates_every_layer_on_two_ranks(tmp_path):
    assert _on_two_ranks(tmp_path, _train_both_ways) == ["True", "True"]


def test_hooks_of_every_norm_run(on_the_host):
    head, seen = _head(), []
    for i, norm in enumerate(head.norm):
        norm.register_forward_hook(lambda *_, i=i: seen.append(i))
    head(torch.randn(3, 12))
    assert seen == [0, 1, 2]


# ---- recomputation ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_head_has_the_gradients_of_its_masks(on_the_host, reentrant):
    a = _head(dropout=0.5)
    b = copy.deepcopy(a)
    xs = [torch.randn(6, 12, requires_grad=True) for _ in range(3)]
    # three calls before the first backward pass, and another one behind it
    outs = [checkpoint(a, x, use_reentrant=reentrant) for x in xs]
    wants = [b(x) for x in xs]
    for out, want in reversed(list(zip(outs, wants))):
        assert torch.equal(out, want)
        out.square().sum().backward()
        want.square().sum().backward()
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(a.parameters(), b.parameters()))
    assert torch.equal(a(xs[0]), b(xs[0])) and [d.calls for d in a.drop] == [d.calls for d in b.drop] == [4, 4]


@pytest.mark.parametrize("reentrant", [False, True])
def test_one_layer_in_several_recomputed_parts(on_the_host, reentrant):
    drop = ldn.Dropout(0.5, seed=3)
    plain = copy.deepcopy(drop)
    x = torch.randn(5, 8, requires_grad=True)
    other = x.detach().clone().requires_grad_()
    y, want = x, other
    for _ in range(3):
        y = checkpoint(lambda v: drop(v * 2), y, use_reentrant=reentrant)
        want = plain(want * 2)
    g = torch.randn(5, 8)
    y.backward(g)
    want.backward(g)
    assert torch.equal(y, want) and torch.equal(x.grad, other.grad)


def test_recomputation_without_the_generators_state_is_refused(on_the_host):
    drop = ldn.Dropout(0.5, seed=3)
    x = torch.randn(5, 8, requires_grad=True)
    y = checkpoint(lambda v: drop(v).square(), x, use_reentrant=False, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match="preserve_rng_state"):
        y.sum().backward()


def test_calls_that_recomputation_cannot_tell_apart_are_refused(on_the_host):
    drop = ldn.Dropout(0.5, seed=3)
    plain = copy.deepcopy(drop)
    x = torch.randn(5, 8, requires_grad=True)

    def seeded():
        torch.manual_seed(1)
        return checkpoint(lambda v: drop(v).square(), x, use_reentrant=False).sum()
    for _ in range(3):  # a generator seeded anew for every step
        got, = torch.autograd.grad(seeded(), x)
        assert torch.equal(got, torch.autograd.grad(plain(x).square().sum(), x)[0])
    first, second = seeded(), seeded()
    for y in (first, second):
        with pytest.raises(RuntimeError, match="same state"):
            torch.autograd.grad(y, x)


def test_a_model_that_cannot_be_quantized_stays_as_it_is():
    model = ldn.ResidualModel(4, 12, [1, 2, 2], hidden=20)
    with pytest.raises(RuntimeError, match="CUDA"):
        model.quantize()
    assert not model._integers and not model._answer


# ---- masks of ranks -------------------------------------------------------------------------------------------------------------------
def _draws(rank):
    drop = ldn.Dropout(0.5, seed=1 + rank)
    drop.draw()
    drop.load_state_dict({"_extra_state": dict(seed=5, calls=3)})  # (one checkpoint for all ranks)
    return [drop.draw() for _ in range(2)]


def test_ranks_with_one_seed_draw_masks_of_their_own(tmp_path):
    first, second = (eval(s) for s in _on_two_ranks(tmp_path, _draws))
    assert first == [(5, 3), (5, 4)]
    assert [seed for seed, _ in second] == [5, 5] and not {o for _, o in first} & {o for _, o in second}
    assert all(0 <= o < 1 << 64 for _, o in second)


# ---- sizes whose sums with a tile's or a grid's would pass 32 bits (none of these calls may launch anything) -----------------------------
MOST = (1 << 31) - 1


@pytest.mark.parametrize("C", [MOST, MOST - 255, MOST - (1 << 22) + 1])
def test_rows_that_are_too_long(C):
    here = ctypes.create_string_buffer(64)
    p = ctypes.cast(here, ctypes.c_void_p)
    assert lib.ldn_layer_norm(p, C, 2, C, 0, p, p, 0, 1e-5, p, p, p, None) == BAD
    assert lib.ldn_layer_norm_backward(p, p, C, 2, C, 0, p, p, p, 0, p, p, p, None) == BAD
    assert lib.ldn_dropout_add_layer_norm(p, C, p, C, 2, C, 0, p, p, 0, 1e-5, 0.5, 1, 0, None, p, p, p, p, None) == BAD
    assert lib.ldn_dropout_add_layer_norm_backward(p, p, p, 2, C, 0, p, p, p, 0, 0.5, 1, 0, None, p, p, p, p, None) == BAD
    assert lib.ldn_quantize_rows(p, C, 2, C, 0, p, C + 16, p, None) == BAD
    assert lib.ldn_layer_norm_quantized(p, C, 2, C, 0, p, p, 0, 1e-5, p, C + 16, p, None) == BAD


@pytest.mark.parametrize("N", [MOST, MOST - 127, MOST - (1 << 22) + 1])
def test_too_many_outputs(N):
    here = ctypes.create_string_buffer(64)
    p = ctypes.cast(here, ctypes.c_void_p)
    assert lib.ldn_int8_linear(p, 16, p, p, 16, p, None, 2, N, 4, 0, p, 0, None) == BAD
    assert lib.ldn_int8_linear_float(p, 16, 0, p, 16, p, None, 2, N, 4, 0, p, 0, None) == BAD
