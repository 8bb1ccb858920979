"""The gated projection on a B200 against the formula in 64 bits."""
import pytest
import torch

import gated_oracle as oracle
import head_oracle
import l_inf_dist_net_v2_b200 as ldn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def made(T, K, H, dtype, seed=0, params=None, biases=(True, True)):
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    x = torch.randn(T, K, **f).to(dtype)
    wg, wu = [(torch.randn(H, K, **f) / K ** 0.5).to(dtype) for _ in range(2)]
    bg, bu = [(0.5 * torch.randn(H, **f)).to(params or dtype) if there else None for there in biases]
    return x, wg, wu, bg, bu, torch.randn(T, H, **f).to(dtype)


def check(x, wg, wu, bg, bu, dy, name):
    dtype = x.dtype
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, wg, wu, bg, bu)]
    y = ldn.gated_linear(*leaves, activation=name)
    f = oracle.forward(x, wg, wu, bg, bu, name, dtype)
    assert y.shape == dy.shape and y.dtype == dtype
    assert head_oracle.near(y.detach().flatten(0, -2), f["y"], f["off_y"])
    with torch.no_grad():
        assert torch.equal(ldn.gated_linear(x, wg, wu, bg, bu, activation=name), y)
    wanted = [t for t in leaves if t is not None]
    got = dict(zip([k for k, t in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), leaves) if t is not None], torch.autograd.grad(y, wanted, dy)))
    for key, (want, bound) in oracle.backward(dy, x, wg, wu, f, name, dtype).items():
        if key in got:
            g = got[key].flatten(0, -2) if key == "x" else got[key]
            assert head_oracle.near(g, want, bound), key


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T, K, H", [(1, 8, 8), (3, 40, 24), (9, 64, 128), (17, 129, 65), (64, 256, 130), (130, 72, 300), (257, 520, 129),
                                     (300, 1000, 520), (20, 5119, 513), (600, 2048, 1100), (1000, 10, 10), (1, 5120, 1025), (33, 1, 1)])
def test_sizes(T, K, H, dtype):
    check(*made(T, K, H, dtype), "silu")
