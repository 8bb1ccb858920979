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
                                     (300, 1000, 520), (20, 5119, 513), (600, 2048, 1100), (1000, 10, 10), (1, 5120, 1025), (33, 1, 1),
                                     (2, 1000, 7), (16, 777, 50), (5, 24, 1), (520, 64, 4100), (4099, 40, 33)])
def test_sizes(T, K, H, dtype):
    check(*made(T, K, H, dtype), "silu")


@pytest.mark.parametrize("name", ["gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T, K, H", [(2, 64, 40), (70, 200, 150), (300, 136, 264)])
def test_activations(T, K, H, dtype, name):
    check(*made(T, K, H, dtype), name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("biases", [(False, False), (True, False), (False, True)])
def test_biases_of_32_bits_and_absent_ones(dtype, biases):
    for T in (3, 90):
        check(*made(T, 96, 72, dtype, params=torch.float32, biases=biases), "silu")
        check(*made(T, 96, 72, dtype, biases=biases), "gelu")


def laid_out(t, layout):
    if layout == "slice":
        return torch.nn.functional.pad(t, (0, 5))[:, :t.size(1)]
    if layout == "wide":
        return torch.nn.functional.pad(t, (0, 16))[:, :t.size(1)]
    if layout == "shifted":
        flat = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)
    if layout == "transposed":
        return t.t().contiguous().t()
    return t[:, None].expand(-1, 2, -1)[:, 0]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["slice", "wide", "shifted", "transposed", "one of two"])
@pytest.mark.parametrize("T", [2, 4, 70])
def test_layouts(T, layout, dtype):
    x, wg, wu, bg, bu, dy = made(T, 104, 50, dtype)
    check(laid_out(x, layout), wg, wu, bg, bu, dy, "silu")
    check(x, laid_out(wg, layout), wu, bg, bu, laid_out(dy, layout), "silu")
    check(x, wg, laid_out(wu, layout), bg, bu, dy, "silu")


def test_shapes():
    x, wg, wu, bg, bu, dy = made(12, 40, 24, torch.float32)
    want = ldn.gated_linear(x, wg, wu, bg, bu)
    assert torch.equal(ldn.gated_linear(x.view(3, 4, 40), wg, wu, bg, bu), want.view(3, 4, 24))
    assert torch.equal(ldn.gated_linear(x[0], wg, wu, bg, bu), ldn.gated_linear(x[:1], wg, wu, bg, bu)[0])
    one = torch.randn(1, 40, device="cuda")[:, ::1].expand(9, 40)
    assert torch.equal(ldn.gated_linear(one, wg, wu), ldn.gated_linear(one.contiguous(), wg, wu))
    for dtype in TYPES:
        leaves = [t.to(dtype).requires_grad_() for t in (x[:0], wg, wu, bg, bu)]
        y = ldn.gated_linear(*leaves)
        grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
        assert y.shape == (0, 24) and grads[0].shape == (0, 40) and not any(g.any() for g in grads[1:])


@pytest.mark.parametrize("T", [3, 200])
def test_gradients_that_are_asked_for_one_by_one(T):
    for dtype in TYPES:
        x, wg, wu, bg, bu, dy = made(T, 64, 48, dtype)
        leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
        whole = torch.autograd.grad(ldn.gated_linear(*leaves), leaves, dy)
        for i, t in enumerate(leaves):
            alone = [s if s is t else s.detach() for s in leaves]
            assert torch.equal(torch.autograd.grad(ldn.gated_linear(*alone), t, dy)[0], whole[i])


def test_gradient_against_differences():
    x, wg, wu, bg, bu, dy = made(6, 24, 16, torch.float32)
    for name in ("silu", "gelu", "sigmoid", "relu"):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu)]
        grads = torch.autograd.grad(ldn.gated_linear(*leaves, activation=name), leaves, dy)
        for i, g in enumerate(grads):
            step = torch.randn_like(g)
            at = [[t.detach() + (s * 2 ** -9 * step if k == i else 0) for k, t in enumerate(leaves)] for s in (1, -1)]
            up, down = [(oracle.forward(*a, name, torch.float32)["y"] * dy.double()).sum() for a in at]
            if name == "relu" and i in (0, 1, 3):  # (steps over a border count as far as the line on either side of it)
                continue
            # (third derivatives of the functions are 1 at most: 2^-18 of the size of the gradients)
            assert abs((up - down) / 2 ** -8 - (g.double() * step).sum()) <= 2.0 ** -14 * (g.double().abs() * step.abs()).sum()


def test_differentiated_twice_says_so():
    x, wg, wu, bg, bu, dy = made(20, 24, 16, torch.float32)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    for wanted in leaves:
        g, = torch.autograd.grad((ldn.gated_linear(*leaves) * dy).sum(), wanted, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            g.square().sum().backward()


@pytest.mark.parametrize("T", [3, 150])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_that_are_not_finite_stay_by_themselves(T, dtype):
    x, wg, wu, bg, bu, dy = made(T, 72, 40, dtype)
    want = ldn.gated_linear(x, wg, wu, bg, bu)
    bad = x.clone()
    bad[1, 5] = float("nan")
    bad[0, 3] = float("inf")
    got = ldn.gated_linear(bad, wg, wu, bg, bu)
    assert got[1].isnan().all() and torch.equal(got[2:], want[2:])
    if T > 8:
        assert not got[0].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_operands_of_all_sizes(dtype):
    """Numbers that need each image of a 32-bit operand, from the smallest to the largest."""
    x, wg, wu, bg, bu, dy = made(40, 136, 72, dtype)
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    small, large = (-60, 60) if dtype != torch.float16 else (-6, 4)
    scale = torch.pow(2.0, torch.randint(small, large, (40, 1), **f).float())
    x = (x.float() * scale).to(dtype)
    want = oracle.forward(x, wg, wu, None, None, "sigmoid", dtype)
    got = ldn.gated_linear(x, wg, wu, activation="sigmoid")
    assert head_oracle.near(got, want["y"], want["off_y"])
    if dtype == torch.float32:  # (the largest numbers are rounded towards zero in their first image)
        one = torch.full((20, 8), torch.finfo(dtype).max, device="cuda")
        eye = torch.eye(8, device="cuda")
        assert torch.equal(ldn.gated_linear(one, eye, eye * 0.5, activation="sigmoid"), one * 0.5)


def test_it_repeats_itself():
    for dtype in TYPES:
        case = made(700, 520, 264, dtype)
        leaves = [t.requires_grad_() for t in case[:5]]
        runs = [(lambda y: (y.detach(),) + torch.autograd.grad(y, leaves, case[5]))(ldn.gated_linear(*leaves)) for _ in range(3)]
        assert all(torch.equal(s, t) for r in runs[1:] for s, t in zip(runs[0], r))


def test_offsets_beyond_32_bits():
    T, K, H = 70001, 16, 32768
    x, wg, wu, bg, bu, _ = made(T, K, H, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    y = ldn.gated_linear(*leaves)
    dy = torch.zeros_like(y)
    dy[-3:] = torch.randn(3, H, device="cuda").bfloat16()
    f = oracle.forward(x[-3:], wg, wu, bg, bu, "silu", torch.bfloat16)
    assert head_oracle.near(y[-3:].detach(), f["y"], f["off_y"])
    gx, gw = torch.autograd.grad(y, (x, wg), dy)
    exact = oracle.backward(dy[-3:], x[-3:], wg, wu, f, "silu", torch.bfloat16)
    assert head_oracle.near(gx[-3:], *exact["x"]) and not gx[:-3].any() and head_oracle.near(gw, *exact["w_gate"])


def test_refusals():
    x, wg, wu, bg, bu, _ = made(4, 8, 6, torch.float32)
    refused = [
        lambda: ldn.gated_linear(x.double(), wg, wu), lambda: ldn.gated_linear(x, wg.half(), wu.half()), lambda: ldn.gated_linear(x, wg, wu[:5]),
        lambda: ldn.gated_linear(x[:, :7], wg, wu), lambda: ldn.gated_linear(x, wg[0], wu[0]), lambda: ldn.gated_linear(x, wg.cpu(), wu),
        lambda: ldn.gated_linear(x, wg, wu, bg[:5]), lambda: ldn.gated_linear(x, wg, wu, bg.half()), lambda: ldn.gated_linear(x, wg, wu, bg.double()),
        lambda: ldn.gated_linear(x.half(), wg.half(), wu.half(), bg.half(), bu), lambda: ldn.gated_linear(x, wg[:0], wu[:0]),
        lambda: ldn.gated_linear(x[:, :0], wg[:, :0], wu[:, :0]), lambda: ldn.gated_linear(x[0, 0], wg, wu),
        lambda: torch.vmap(lambda t: ldn.gated_linear(t, wg, wu))(x[None]),
    ]
    before = ldn._lib.lib.ldn_kernel_launches()
    for call in refused:
        with pytest.raises(RuntimeError):
            call()
    assert ldn._lib.lib.ldn_kernel_launches() == before


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("step", [0, 1, 3, 7, 8, 13])
@pytest.mark.parametrize("T, K", [(5, 40), (70, 104), (9, 99), (300, 16)])
def test_rows_that_are_repeated_or_overlap(T, K, step, dtype):
    _, wg, wu, bg, bu, dy = made(T, K, 24, dtype)
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(step))
    for start in (0, 3):
        flat = torch.randn(start + (T - 1) * step + K, **f).to(dtype)[start:]
        x = flat[:K].expand(T, K) if step == 0 else flat.unfold(0, K, step)
        assert x.shape == (T, K) and x.stride() == (step, 1)
        runs = []
        for rows in (x, x.contiguous()):
            leaves = [t.detach().requires_grad_() for t in (rows, wg, wu, bg, bu)]
            y = ldn.gated_linear(*leaves)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("step", [0, 1, 8])
@pytest.mark.parametrize("T, K", [(1, 40), (3, 1), (70, 104), (20, 16), (33, 1)])
def test_weights_whose_rows_are_repeated_or_overlap(T, K, step, dtype):
    x, wg, wu, bg, bu, dy = made(T, K, 24, dtype)
    flat = torch.randn(23 * step + K, device="cuda").to(dtype)
    w = flat.expand(24, K) if step == 0 else flat.unfold(0, K, step)
    assert w.shape == (24, K)
    for one, other in ((w, wu), (wg, w), (w, w)):
        runs = []
        for a, b in ((one, other), (one.contiguous(), other.contiguous())):
            leaves = [t.detach().requires_grad_() for t in (x, a, b, bg, bu)]
            y = ldn.gated_linear(*leaves)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
        assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert ldn.gated_linear(x, w[:1], w[:1]).shape == (T, 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T, K, H", [(16385, 72, 40), (20000, 200, 300), (40, 16400, 72), (300, 20001, 130), (24, 40, 8193), (300, 72, 10000)])
def test_sums_of_more_terms_than_stay_in_the_accumulator(T, K, H, dtype):
    check(*made(T, K, H, dtype), "silu")


# (sums leave the accumulator after 4096 terms: 256 instructions that drop less than 2^-23 of it each; then they are added up in 32 bits, and so
# are the parts of a tile that several pairs of CTAs share)
def drained(terms):
    return 256 * 2.0 ** -23 + (terms / 4096 + 80) * head_oracle.EPS32


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_long_sums_are_not_smaller_for_it(dtype):
    """Sums of positive products alone, with relu of one as the gate: y = u, du = dy and dg = dy u exactly where u is a power of two."""
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    T, C = 262144, 2048
    x, dy = (torch.rand(T, C, **f) + 0.5).to(dtype), ((torch.rand(T, C, **f) + 0.5) * 2.0 ** -6).to(dtype)
    zero, one = torch.zeros(C, C, device="cuda", dtype=dtype), torch.ones(C, device="cuda", dtype=dtype)
    wu = zero.clone().requires_grad_()
    got, = torch.autograd.grad(ldn.gated_linear(x, zero, wu, one, one, activation="relu"), wu, dy)
    want = torch.cat([dy[:, i:i + 8].double().t() @ x.double() for i in range(0, 64, 8)])
    assert head_oracle.near(got[:64], want, drained(T) * want)
    del x, dy, got
    T, K, H = 600, 131072, 1100
    x, wu = (torch.rand(T, K, **f) + 0.5).to(dtype), ((torch.rand(H, K, **f) + 0.5) * 2.0 ** -7).to(dtype)
    got = ldn.gated_linear(x, torch.zeros_like(wu), wu, torch.ones(H, device="cuda", dtype=dtype), activation="relu")
    want = x[:64].double() @ wu.double().t()
    assert head_oracle.near(got[:64], want, (drained(K) + 4 * head_oracle.EPS32) * want)
    T, K, H = 300, 600, 131072
    dy, w = ((torch.rand(T, H, **f) + 0.5) * 2.0 ** -7).to(dtype), (torch.rand(H, K, **f) + 0.5).to(dtype)
    x, one = torch.zeros(T, K, device="cuda", dtype=dtype, requires_grad=True), torch.ones(H, device="cuda", dtype=dtype)
    got, = torch.autograd.grad(ldn.gated_linear(x, w, w, one, one, activation="relu"), x, dy)
    want = 2 * dy[:64].double() @ w.double()
    assert head_oracle.near(got[:64], want, drained(2 * H) * want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T", [1, 40])
def test_gelu_keeps_its_digits_far_below_zero(T, dtype):
    """The gate is a bias alone, so that the function and its slope come by themselves.  The normal distribution's function is off by a dozen units
    of itself, e^(-g^2 / 2) by eight; products and sums round once each (and a bias's gradient T / 8 + 64 times)."""
    g = torch.cat([torch.linspace(-14, 10, 8000), torch.tensor([-0.0, 0.0, -30.0, 30.0, 1e30, -1e30])]).cuda()
    H, unit, least = g.numel(), head_oracle.EPS32, 64 * 2.0 ** -149
    x, w, one = torch.zeros(T, 8, device="cuda", dtype=dtype), torch.zeros(H, 8, device="cuda", dtype=dtype), torch.ones(H, device="cuda")
    leaf = g.clone().requires_grad_()
    y = ldn.gated_linear(x, w, w, leaf, one, activation="gelu")
    got, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    g = g.double()
    cdf = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
    bell = g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    want = (g * cdf).expand(T, H)
    held = want.abs() <= torch.finfo(dtype).max  # (1e30 is infinity in float16)
    assert head_oracle.near(y.detach()[held], want[held], 16 * unit * want[held].abs() + least)
    assert (y.detach()[~held] == float("inf")).all() and (dtype == torch.float16 or held.all())
    bound = unit * (16 * cdf + 12 * bell.abs() + (T / 8 + 64) * (T > 1) * (cdf + bell).abs()) + least
    assert head_oracle.near(got, T * (cdf + bell), T * bound)
    ends = torch.tensor([float("inf"), float("nan")], device="cuda")
    y = ldn.gated_linear(x, w[:2], w[:2], ends, one[:2], activation="gelu")
    assert (y[:, 0] == float("inf")).all() and y[:, 1].isnan().all()


@pytest.mark.parametrize("T", [1, 40])
def test_the_slope_of_a_gate_that_is_wide_open_keeps_its_digits(T):
    """As for gelu; s and 1 - s are off by eight units of themselves, their product by two more."""
    g, unit = torch.linspace(-80, 80, 8001).cuda(), head_oracle.EPS32
    H = g.numel()
    x, w, one = torch.zeros(T, 8, device="cuda"), torch.zeros(H, 8, device="cuda"), torch.ones(H, device="cuda")
    chain = 18 + (T / 8 + 64) * (T > 1)
    e = torch.exp(-g.double().abs())
    s = torch.where(g < 0, e, 1.0) / (1 + e)
    rest = torch.where(g < 0, 1.0, e) / (1 + e)
    for name, want, size in (("sigmoid", s * rest, s * rest), ("silu", s * (1 + g.double() * rest), s * (1 + g.double().abs() * rest))):
        leaf = g.clone().requires_grad_()
        got, = torch.autograd.grad(ldn.gated_linear(x, w, w, leaf, one, activation=name).sum(), leaf)
        assert head_oracle.near(got, T * want, T * chain * unit * size), name
