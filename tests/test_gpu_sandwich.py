"""The residual stream between two norms on a B200 against the formulas in 64 bits."""
import pytest
import torch

import head_oracle
import l_inf_dist_net_v2_b200 as ldn
import sandwich_oracle as oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
# one element; fewer than a 16-byte piece; around a warp's and a block's reach; odd; the longest of each way, and beyond
LENGTHS = [1, 3, 8, 31, 96, 128, 257, 512, 1000, 1001, 1024, 4097, 5120, 5121, 8192, 16384, 20000]
NAMES = ["x", "residual", "gate", "scale", "pw", "pb", "w", "b"]


def _rows(rows, C, dtype, f, layout):
    x = (torch.randn(rows, C, **f) * (torch.rand(rows, 1, **f) * 2 + 0.5) + torch.randn(rows, 1, **f)).to(dtype)
    if layout == "slice":
        return torch.nn.functional.pad(x, (0, 5))[:, :C]
    if layout == "shifted":
        flat = torch.empty(rows * C + 1, device="cuda", dtype=dtype)
        flat[1:] = x.view(-1)
        return flat[1:].view(rows, C)
    return x


def made(rows, C, dtype, gate="none", params=None, layout="plain", absent=(), seed=0):
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 100 * C))
    p = params or dtype
    t = dict(x=_rows(rows, C, dtype, f, layout), residual=_rows(rows, C, dtype, f, layout), gate=None)
    if gate != "none":
        t["gate"] = _rows(rows, 1 if gate == "row" else C, dtype, f, layout if gate == "all" else "plain").sigmoid()
    for name, one in (("scale", 0.5), ("pw", 1.0), ("pb", 0.0), ("w", 1.0), ("b", 0.0)):
        t[name] = None if name in absent else (one + 0.3 * torch.randn(C, **f)).to(p)
    return t, torch.randn(rows, C, **f).to(dtype), torch.randn(rows, C, **f).to(dtype)


def call(t, eps=1e-5):
    return ldn.sandwich_norm(t["x"], t["residual"], t["w"], t["b"], t["pw"], t["pb"], t["scale"], t["gate"], eps)


def check(t, dy, dh, use=("y", "h")):
    t = {k: v if v is None else v.detach().requires_grad_() for k, v in t.items()}
    y, h = call(t)
    held = {k: v if v is None else v.detach() for k, v in t.items()}
    assert y.dtype == h.dtype == held["x"].dtype and y.is_contiguous() and h.is_contiguous()
    want, bound = oracle.forward(*[held[k] for k in ("x", "residual", "gate", "scale", "pw", "pb")], 1e-5)
    assert head_oracle.near(h.detach(), want, bound), "h"
    want, _, _, _, bound = head_oracle.norm(h.detach(), held["w"], held["b"], 1e-5)
    assert head_oracle.near(y.detach(), want, bound), "y"
    with torch.no_grad():
        again = call(t)
        assert torch.equal(again[0], y) and torch.equal(again[1], h)
    wanted = {k: v for k, v in t.items() if v is not None}
    outs, ups = zip(*[(o, u) for n, o, u in (("y", y, dy), ("h", h, dh)) if n in use])
    got = dict(zip(wanted, torch.autograd.grad(outs, list(wanted.values()), ups, allow_unused=True)))
    exact = oracle.backward(dy if "y" in use else None, dh if "h" in use else None, held["x"], h.detach(), held["gate"], held["scale"], held["pw"],
                            held["pb"], held["w"], 1e-5)
    for name, g in got.items():
        want, bound = exact[name]
        assert g.shape == t[name].shape and g.dtype == t[name].dtype
        assert head_oracle.near(g, want.view_as(g), bound.view_as(g)), name


@pytest.mark.parametrize("gate", ["none", "row", "all"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("C", LENGTHS)
def test_lengths(C, dtype, gate):
    rows = 3 if C > 10000 else 37
    for layout, params in [("plain", F32), ("plain", dtype), ("slice", F32), ("shifted", dtype)]:
        check(*made(rows, C, dtype, gate, params, layout))


@pytest.mark.parametrize("rows, C", [(1, 96), (5000, 96), (1000, 1000), (700, 5120), (3001, 33)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_rows(rows, C, dtype):
    for gate in ("row", "all"):
        check(*made(rows, C, dtype, gate, F32))


@pytest.mark.parametrize("absent", [("scale",), ("pw", "pb"), ("w", "b"), ("pb", "b", "scale"), ("scale", "pw", "pb", "w", "b")])
@pytest.mark.parametrize("C", [96, 1001, 6000])
def test_absent_parameters(C, absent):
    for dtype in TYPES:
        check(*made(40, C, dtype, "row", F32, absent=absent))


@pytest.mark.parametrize("use", [("y",), ("h",)])
@pytest.mark.parametrize("C", [96, 1024, 6000])
def test_one_gradient_comes(C, use):
    for dtype in (F32, BF16):
        check(*made(33, C, dtype, "all", F32), use=use)
