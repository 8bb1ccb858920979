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


def test_shapes_strides_and_no_rows():
    t, dy, dh = made(12, 40, F32, "row")
    y, h = call(t)
    cube = {k: v.view(3, 4, -1) if k in ("x", "residual", "gate") else v for k, v in t.items()}
    for got, want in zip(call(cube), (y, h)):
        assert torch.equal(got, want.view(3, 4, 40))
    turned = {k: v.t().contiguous().t() if k in ("x", "residual", "gate") else v for k, v in t.items()}
    for got, want in zip(call(turned), (y, h)):
        assert torch.equal(got, want)
    for dtype in TYPES:
        for gate in ("none", "row", "all"):
            t, _, _ = made(3, 40, dtype, gate)
            t = {k: v if v is None else (v[:0] if k in ("x", "residual", "gate") else v).detach().requires_grad_() for k, v in t.items()}
            wanted = [v for v in t.values() if v is not None]
            y, h = call(t)
            grads = torch.autograd.grad((y, h), wanted, (torch.empty_like(y), torch.empty_like(h)))
            assert y.shape == h.shape == (0, 40) and not any(g.any() for g in grads)


@pytest.mark.parametrize("C", [40, 1024])
def test_gradients_that_are_asked_for_one_by_one(C):
    for gate in ("row", "all"):
        t, dy, dh = made(30, C, BF16, gate, F32)
        t = {k: v.requires_grad_() for k, v in t.items()}
        whole = torch.autograd.grad(call(t), list(t.values()), (dy, dh))
        for name, g in zip(t, whole):
            alone = {k: v if k == name else v.detach() for k, v in t.items()}
            if name in ("w", "b"):
                got, = torch.autograd.grad(call(alone)[0], alone[name], dy)
            else:
                got, = torch.autograd.grad(call(alone), alone[name], (dy, dh))
            assert torch.equal(got, g), name


def test_gradient_against_differences():
    for gate in ("none", "row", "all"):
        t, dy, dh = made(5, 24, F32, gate)
        leaves = {k: v.double().requires_grad_() for k, v in t.items() if v is not None}
        grads = dict(zip(leaves, torch.autograd.grad(call({k: v.float() if v is not None else None for k, v in {**t, **leaves}.items()}),
                                                      list(leaves.values()), (dy, dh))))

        def value(at):
            h, _ = oracle.forward(*[at.get(k) for k in ("x", "residual", "gate", "scale", "pw", "pb")], 1e-5)
            y = head_oracle.norm(h, at.get("w"), at.get("b"), 1e-5)[0]
            return (y * dy.double()).sum() + (h * dh.double()).sum()
        for name, g in grads.items():
            step = torch.randn_like(leaves[name])
            up, down = (value({k: v.detach() + (s * 2 ** -10 * step if k == name else 0) for k, v in leaves.items()}) for s in (1, -1))
            size = sum((v.abs() * torch.ones_like(v)).sum() for v in (g.abs() * step.abs(),)) + dy.double().abs().sum()
            assert abs((up - down) / 2 ** -9 - (g * step).sum()) <= 2.0 ** -14 * size, name


def test_differentiated_twice_says_so():
    t, dy, dh = made(6, 40, F32, "row")
    t = {k: v.requires_grad_() for k, v in t.items()}
    for name in ("x", "residual", "gate", "scale", "pw", "w"):
        y, _ = call(t)
        g, = torch.autograd.grad((y * dy).sum(), t[name], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            g.square().sum().backward()


@pytest.mark.parametrize("C", [8, 96, 1001, 4096, 6001])
def test_rows_that_are_constant_large_or_not_finite(C):
    t, dy, dh = made(9, C, F32, "row", layout="plain")
    t["x"][0] = 3.0             # (nothing but the first norm's bias joins the stream)
    t["x"][1] *= 1e15
    t["residual"][2] += 1e6
    t["x"][3, 0] = float("nan")
    t["residual"][4, C // 2] = float("inf")
    t["gate"][5] = 0.0
    t = {k: v.requires_grad_() for k, v in t.items()}
    y, h = call(t)
    held = {k: v.detach() for k, v in t.items()}
    want, bound = oracle.forward(*[held[k] for k in ("x", "residual", "gate", "scale", "pw", "pb")], 1e-5)
    good = [0, 1, 2, 5, 6, 7, 8]
    assert head_oracle.near(h.detach()[good], want[good], bound[good])
    assert torch.equal(h[5], held["residual"][5]) and y[[3, 4]].isnan().any(1).all() and y[good].isfinite().all()
    gx, gr = torch.autograd.grad((y, h), (t["x"], t["residual"]), (dy, dh))
    assert gx[good].isfinite().all() and gr[good].isfinite().all() and not gx[5].any()


def test_offsets_beyond_32_bits():
    rows, C = 300000, 8000
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    t = {k: torch.empty(rows, C, device="cuda", dtype=BF16).normal_(generator=f["generator"]) for k in ("x", "residual")}
    t["gate"] = torch.rand(rows, 1, **f).to(BF16)
    t.update({k: torch.randn(C, **f) for k in ("scale", "pw", "pb", "w", "b")})
    t = {k: v.requires_grad_() for k, v in t.items()}
    dy, dh = torch.zeros(2, rows, C, device="cuda", dtype=BF16)
    dy[-5:], dh[-5:] = torch.randn(2, 5, C, **f)
    y, h = call(t)
    grads = dict(zip(t, torch.autograd.grad((y, h), list(t.values()), (dy, dh))))
    few = {k: (v[-5:] if v.size(0) == rows else v).detach().requires_grad_() for k, v in t.items()}
    y5, h5 = call(few)
    want = dict(zip(few, torch.autograd.grad((y5, h5), list(few.values()), (dy[-5:], dh[-5:]))))
    assert torch.equal(y[-5:], y5) and torch.equal(h[-5:], h5)
    for name, g in grads.items():
        if g.size(0) == rows:
            assert torch.equal(g[-5:], want[name])
        else:
            assert torch.allclose(g, want[name], rtol=1e-5, atol=1e-5 * want[name].abs().max().item())


def test_refusals():
    t, _, _ = made(4, 8, F32, "row")
    x, r, g, w = t["x"], t["residual"], t["gate"], t["w"]
    refused = [
        lambda: ldn.sandwich_norm(x.double(), r), lambda: ldn.sandwich_norm(x, r[:3]), lambda: ldn.sandwich_norm(x, r.half()),
        lambda: ldn.sandwich_norm(x, r, w[:7]), lambda: ldn.sandwich_norm(x, r, w.half()), lambda: ldn.sandwich_norm(x, r, w.cpu()),
        lambda: ldn.sandwich_norm(x.half(), r.half(), w.half(), post_weight=w), lambda: ldn.sandwich_norm(x, r, gate=g[:, 0]),
        lambda: ldn.sandwich_norm(x, r, gate=g.half()), lambda: ldn.sandwich_norm(x, r, gate=torch.ones(4, 3, device="cuda")),
        lambda: ldn.sandwich_norm(x, r, eps=-1.0), lambda: ldn.sandwich_norm(x[:, :0], r[:, :0]), lambda: ldn.sandwich_norm(x, r, scale=w[None]),
        lambda: torch.vmap(lambda a: ldn.sandwich_norm(a, a)[0])(x[None]),
    ]
    before = ldn._lib.lib.ldn_kernel_launches()
    for attempt in refused:
        with pytest.raises(RuntimeError):
            attempt()
    assert ldn._lib.lib.ldn_kernel_launches() == before


@pytest.mark.parametrize("rows, C", [(300, 5121), (200, 8192), (150, 10975), (130, 16385), (100, 33000), (20, 40960), (5, 41001)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_rows_that_blocks_share(rows, C, dtype):
    for gate in ("none", "row", "all"):
        check(*made(rows, C, dtype, gate, F32 if gate == "row" else dtype))
    check(*made(rows, C, dtype, "all", F32, layout="shifted"), use=("y",))


@pytest.mark.parametrize("gate", ["none", "row", "all"])
@pytest.mark.parametrize("C, layout", [(96, "plain"), (33, "plain"), (1024, "plain"), (4097, "plain"), (16384, "plain"), (60000, "plain"), (520, "shifted")])
def test_without_the_gradient_of_y_it_does_not_matter_what_h_is(C, layout, gate):
    """h with infinities and what is not a number: the gradients of h alone are those of any other h."""
    for dtype in TYPES:
        t, _, dh = made(9, C, dtype, gate, F32, layout)
        held = {k: v if v is None else v.detach() for k, v in t.items()}
        want = oracle.backward(None, dh, held["x"], held["x"], held["gate"], held["scale"], held["pw"], held["pb"], held["w"], 0.0)
        t["residual"] = t["residual"].clone()
        t["residual"][2, C // 2], t["residual"][4, 0], t["residual"][5, C - 1] = float("inf"), float("-inf"), float("nan")
        t = {k: v if v is None else v.detach().requires_grad_() for k, v in t.items()}
        h = call(t, 0.0)[1]
        assert not h[2, C // 2].isfinite() and not h[5, C - 1].isfinite()
        leaves = {k: v for k, v in t.items() if v is not None}
        for name, g in zip(leaves, torch.autograd.grad(h, list(leaves.values()), dh)):
            if name in ("w", "b"):
                assert not g.any(), name
            else:
                assert head_oracle.near(g, want[name][0].view_as(g), want[name][1].view_as(g)), name
        assert torch.equal(torch.autograd.grad(call(t, 0.0)[1], t["residual"], dh)[0], dh)


@pytest.mark.parametrize("gate", ["none", "row", "all"])
@pytest.mark.parametrize("rows, C, dtype", [(20003, 1001, F32), (40000, 1024, BF16), (9001, 5120, F16), (90000, 500, F32), (300000, 96, F32),
                                            (5001, 9000, F32)])
def test_without_the_gradient_of_y_of_many_rows(rows, C, dtype, gate):
    """They have the gradients of a y whose gradient is zero."""
    t, _, dh = made(rows, C, dtype, gate, F32)
    t = {k: v if v is None else v.detach().requires_grad_() for k, v in t.items()}
    y, h = call(t)
    leaves = {k: v for k, v in t.items() if v is not None}
    alone = torch.autograd.grad(h, list(leaves.values()), dh, retain_graph=True)
    exact = oracle.backward(None, dh, *[None if v is None else v.detach() for v in (t["x"], h, t["gate"], t["scale"], t["pw"], t["pb"], t["w"])], 1e-5)
    for name, g in zip(leaves, alone):
        want, bound = exact[name]
        assert head_oracle.near(g, want.view_as(g), bound.view_as(g)), name
    both = torch.autograd.grad((y, h), list(leaves.values()), (torch.zeros_like(y), dh))
    for name, g, same in zip(leaves, alone, both):
        if name in ("x", "residual", "gate"):
            assert torch.equal(g, same), name
