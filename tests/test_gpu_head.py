"""Layer norm, dropout, both joined, and the product in 8-bit integers against evaluations in 64 bits (tests/head_oracle.py), at the
lengths, alignments and values where they can go wrong.  Tolerances are bounds on evaluations in 32 bits, derived in the oracle."""
import numpy as np
import pytest
import torch

import head_oracle as oracle
import l_inf_dist_net_v2_b200 as ldn
from l_inf_dist_net_v2_b200._lib import lib

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
# one element; fewer than a 16-byte piece; around a warp's and a block's reach; odd; the longest that registers hold, and beyond
LENGTHS = [1, 3, 8, 31, 96, 128, 257, 512, 1000, 1001, 1024, 4097, 5120, 16384, 20000, 40008]


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _rows(rows, C, dtype, seed, layout="plain"):
    """Activations with a scale and a mean per row: contiguous, as a slice of wider rows, or starting off 16 bytes."""
    f = _gen(seed)
    x = (torch.randn(rows, C, **f) * (torch.rand(rows, 1, **f) * 2 + 0.5) + torch.randn(rows, 1, **f)).to(dtype)
    if layout == "slice":
        return torch.nn.functional.pad(x, (0, 5))[:, :C]
    if layout == "shifted":
        flat = torch.empty(rows * C + 1, device="cuda", dtype=dtype)
        flat[1:] = x.view(-1)
        return flat[1:].view(rows, C)
    return x


def _params(C, dtype, seed):
    f = _gen(seed)
    return (1 + 0.3 * torch.randn(C, **f)).to(dtype), (0.3 * torch.randn(C, **f)).to(dtype)


# ---- layer norm -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", LENGTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm(C, dtype):
    rows = 3 if C > 10000 else 37
    for layout, wide in [("plain", True), ("plain", False), ("slice", True), ("shifted", False)]:
        x = _rows(rows, C, dtype, C, layout).detach().requires_grad_()
        w, b = (t.requires_grad_() for t in _params(C, F32 if wide else dtype, C + 1))
        g = torch.randn(rows, C, **_gen(C + 2)).to(dtype)
        y = ldn.layer_norm(x, w, b, 1e-5)
        assert y.dtype == dtype and y.is_contiguous()
        want, _, _, _, bound = oracle.norm(x.detach(), w.detach(), b.detach(), 1e-5)
        assert oracle.near(y.detach(), want, bound), (layout, wide)
        grads = torch.autograd.grad(y, (x, w, b), g)
        for name, got, (want, bound) in zip("xwb", grads, oracle.norm_grad(g, x.detach(), w.detach(), 1e-5)):
            assert got.dtype == (dtype if name == "x" else w.dtype)
            assert oracle.near(got, want, bound), (name, layout, wide)
        with torch.no_grad():
            assert torch.equal(ldn.layer_norm(x, w, b, 1e-5), y)


@pytest.mark.parametrize("rows", [1, 2, 5, 64, 147, 149, 1000, 5000])
@pytest.mark.parametrize("C, dtype", [(96, BF16), (512, F32), (1001, F16), (5120, BF16)])
def test_norm_over_many_rows(rows, C, dtype):
    x, (w, b) = _rows(rows, C, dtype, rows).requires_grad_(), _params(C, F32, 1)
    w, b = w.requires_grad_(), b.requires_grad_()
    g = torch.randn(rows, C, **_gen(2)).to(dtype)
    y = ldn.layer_norm(x, w, b, 1e-5)
    first = torch.autograd.grad(y, (x, w, b), g, retain_graph=True)
    for got, (want, bound) in zip(first, oracle.norm_grad(g, x.detach(), w.detach(), 1e-5)):
        assert oracle.near(got, want, bound)
    assert all(torch.equal(a, c) for a, c in zip(first, torch.autograd.grad(y, (x, w, b), g)))  # sums in a fixed order


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_norm_with_some_parameters(dtype, which):
    x, (w, b) = _rows(9, 200, dtype, 5).requires_grad_(), _params(200, F32, 6)
    w, b = (w.requires_grad_() if which == "weight" else None), (b.requires_grad_() if which == "bias" else None)
    y = ldn.layer_norm(x, w, b, 1e-3)
    want, _, _, _, bound = oracle.norm(x.detach(), w, b, 1e-3)
    assert oracle.near(y.detach(), want.detach(), bound.detach())
    g = torch.randn(9, 200, **_gen(7)).to(dtype)
    wanted = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, wanted, g)
    exact = oracle.norm_grad(g, x.detach(), None if w is None else w.detach(), 1e-3)
    exact = [exact[0]] + [exact[1]] * (w is not None) + [exact[2]] * (b is not None)
    for got, (want, bound) in zip(grads, exact):
        assert oracle.near(got, want, bound)


def test_norm_gradients_that_are_asked_for_one_by_one():
    x, (w, b) = _rows(33, 300, F32, 5).requires_grad_(), [t.requires_grad_() for t in _params(300, F32, 6)]
    g = torch.randn(33, 300, **_gen(7))
    y = ldn.layer_norm(x, w, b)
    every = torch.autograd.grad(y, (x, w, b), g, retain_graph=True)
    for t, want in zip((x, w, b), every):
        assert torch.equal(torch.autograd.grad(y, t, g, retain_graph=True)[0], want)
    frozen = ldn.layer_norm(x, w.detach(), b)
    assert torch.equal(torch.autograd.grad(frozen, b, g)[0], every[2])


def test_norm_gradient_against_differences():
    x, (w, b) = _rows(5, 64, F32, 11).requires_grad_(), [t.requires_grad_() for t in _params(64, F32, 12)]
    g, h = torch.randn(5, 64, **_gen(13)), 1e-2
    grads = torch.autograd.grad(ldn.layer_norm(x, w, b), (x, w, b), g)
    with torch.no_grad():
        for k, grad in enumerate(grads):
            v = torch.randn(grad.shape, **_gen(14 + k))
            at = lambda s: (ldn.layer_norm(*[t + s * v if i == k else t for i, t in enumerate((x, w, b))]).double() * g).sum()  # noqa: E731
            slope, want = (at(h) - at(-h)) / (2 * h), (grad.double() * v).sum()
            # third derivatives of a row's norm are a few rstd^3 (rstd up to 2.5), and there are 320 terms of size 1
            assert abs(slope - want) <= 320 * (h * h * 20 + 64 * 2.0 ** -24 / h) / 10


@pytest.mark.parametrize("C", [7, 96, 1024, 5120, 40000])
def test_norm_rows_that_are_constant_large_or_not_finite(C):
    x = torch.randn(6, C, **_gen(C))
    x[0] = 3.25
    x[1] = 0
    x[2] = 1e4 + x[2]
    x[3] *= 1e15
    w, b = _params(C, F32, 1)
    want, _, _, _, bound = oracle.norm(x, w, b, 1e-5)
    y = ldn.layer_norm(x, w, b, 1e-5)
    assert oracle.near(y, want, bound)
    bad = x.clone()
    bad[4, C // 2], bad[5, 0] = float("nan"), float("inf")
    got = ldn.layer_norm(bad, w, b, 1e-5)
    assert got[4:].isnan().all() and torch.equal(got[:4], y[:4])


def test_norm_shapes_and_strides():
    f = _gen(3)
    w, b = _params(48, F32, 4)
    for x in (torch.randn(48, **f), torch.randn(2, 3, 5, 48, **f), torch.randn(4, 48, 6, **f).transpose(1, 2),
              torch.randn(7, 6, 48, **f)[:, 2:4], torch.randn(3, 1, 48, **f).expand(3, 5, 48), torch.randn(48, **f).expand(2, 3, 48),
              torch.randn(5, 96, **f)[:, ::2], torch.randn(0, 48, **f)):
        y = ldn.layer_norm(x, w, b)
        assert y.shape == x.shape
        want, _, _, _, bound = oracle.norm(x, w, b, 1e-5)
        assert x.numel() == 0 or oracle.near(y, want, bound)
    x = torch.randn(0, 48, **f).requires_grad_()
    w.requires_grad_()
    gx, gw = torch.autograd.grad(ldn.layer_norm(x, w, b).sum(), (x, w))
    assert gx.shape == (0, 48) and torch.equal(gw, torch.zeros_like(gw))


# ---- dropout --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (1, 4097), (64, 1024), (33, 1001), (257, 96)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_dropout(shape, dtype, p):
    seed, offset = 0x9E3779B97F4A7C15, (1 << 40) + 3
    kept = oracle.keep(shape, p, seed, offset)
    for layout in ("plain", "slice", "shifted"):
        for onto in (False, True):
            x = _rows(*shape, dtype, 5, layout).detach().requires_grad_()
            r = _rows(*shape, dtype, 6, layout).detach().requires_grad_() if onto else None
            out = ldn.dropout(x, p, seed, offset, residual=r)
            want = oracle.dropped(x.detach(), kept, p)
            assert torch.equal(out, (want if r is None else r.detach().float() + want).to(dtype))
            g = torch.randn(shape, **_gen(7)).to(dtype)
            grads = torch.autograd.grad(out, (x, r) if onto else (x,), g)
            assert torch.equal(grads[0], oracle.dropped(g, kept, p).to(dtype))
            assert not onto or torch.equal(grads[1], g)


def test_dropout_is_another_mask_for_another_seed_or_offset():
    x = torch.ones(64, 1024, device="cuda")
    masks = [ldn.dropout(x, 0.5, s, o) != 0 for s, o in [(1, 0), (2, 0), (1, 1), (1 << 32, 0), (1, 1 << 32)]]
    for i, a in enumerate(masks):
        assert abs(a.float().mean().item() - 0.5) < 6 * 0.5 / 256  # six deviations of a mean of 65536
        for b in masks[:i]:
            assert abs((a == b).float().mean().item() - 0.5) < 6 * 0.5 / 256


def test_dropout_with_a_seed_on_the_device():
    x = _rows(40, 100, F32, 1).requires_grad_()
    state = torch.tensor([77, 5], device="cuda")
    out = ldn.dropout(x, 0.3, state, 2)
    assert torch.equal(out, ldn.dropout(x, 0.3, 77, 7))
    state += 1  # the gradient is that of the mask that was drawn
    g = torch.randn(40, 100, **_gen(2))
    assert torch.equal(torch.autograd.grad(out, x, g)[0], oracle.dropped(g, oracle.keep((40, 100), 0.3, 77, 7), 0.3))
    assert torch.equal(ldn.dropout(x, 0.3, state, 2), ldn.dropout(x, 0.3, 78, 8))


def test_dropout_twice_differentiated():
    x = _rows(8, 12, F32, 1).requires_grad_()
    g = torch.randn(8, 12, **_gen(2)).requires_grad_()
    gx, = torch.autograd.grad(ldn.dropout(x, 0.4, 3), x, g, create_graph=True)
    v = torch.randn(8, 12, **_gen(3))
    assert torch.equal(torch.autograd.grad(gx, g, v)[0], oracle.dropped(v, oracle.keep((8, 12), 0.4, 3, 0), 0.4))


def test_dropout_keeps_what_is_not_finite_out_of_dropped_places():
    x = torch.full((4, 64), float("nan"), device="cuda")
    kept = oracle.keep((4, 64), 0.5, 9, 0).cuda()
    assert torch.equal(ldn.dropout(x, 0.5, 9).isnan(), kept)


# ---- both, on a residual stream ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", [1, 5, 96, 130, 512, 1001, 4100, 5120, 16384, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_joined(C, dtype):
    rows, p, seed, offset = (3 if C > 10000 else 41), 0.2, 1234567890123, 9
    kept = oracle.keep((rows, C), p, seed, offset)
    for layout, wide in [("plain", True), ("plain", False), ("slice", True), ("shifted", False)]:
        x, r = (_rows(rows, C, dtype, C + k, layout).detach().requires_grad_() for k in (0, 1))
        w, b = (t.requires_grad_() for t in _params(C, F32 if wide else dtype, C + 2))
        y, h = ldn.dropout_add_layer_norm(x, r, w, b, p, seed, offset)
        want_h = (r.detach().float() + oracle.dropped(x.detach(), kept, p)).to(dtype)
        assert torch.equal(h, want_h)
        want, _, _, _, bound = oracle.norm(want_h, w.detach(), b.detach(), 1e-5)
        assert oracle.near(y.detach(), want, bound)
        gy, gh = (torch.randn(rows, C, **_gen(C + k)).to(dtype) for k in (3, 4))
        gx, gr, gw, gb = torch.autograd.grad((y, h), (x, r, w, b), (gy, gh), retain_graph=True)
        (want_x, off_x), sums_w, sums_b = oracle.norm_grad(gy, want_h, w.detach(), 1e-5)
        whole = want_x + gh.double()
        off = off_x + oracle.EPS32 * whole.abs()
        scale = float(np.float32(1 / (1 - p)))
        assert oracle.near(gr, whole, off)
        assert oracle.near(gx, torch.where(kept.cuda(), whole * scale, 0.0), (off * scale + oracle.EPS32 * whole.abs() * 2))
        assert oracle.near(gw, *sums_w) and oracle.near(gb, *sums_b)
        # the stream alone, and the norm alone
        only_h = torch.autograd.grad(h, (x, r), gh, retain_graph=True)
        assert oracle.near(only_h[1], gh.double(), oracle.EPS32 * gh.double().abs())
        only_y = torch.autograd.grad(y, (x, r), gy)
        assert oracle.near(only_y[1], want_x, off_x)
        with torch.no_grad():
            assert all(torch.equal(s, t) for s, t in zip((y, h), ldn.dropout_add_layer_norm(x, r, w, b, p, seed, offset)))


@pytest.mark.parametrize("p", [0.0, 1.0])
def test_joined_at_the_ends(p):
    x, r, (w, b) = _rows(6, 100, F32, 1), _rows(6, 100, F32, 2), _params(100, F32, 3)
    y, h = ldn.dropout_add_layer_norm(x, r, w, b, p, 4)
    assert torch.equal(h, r + x if p == 0 else r)
    assert oracle.near(y, *[oracle.norm(h, w, b, 1e-5)[i] for i in (0, 4)])


# ---- 8-bit integers -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", LENGTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_as_integers(C, dtype):
    for layout in ("plain", "slice", "shifted"):
        x = _rows(9, C, dtype, C, layout)
        x[0] = 0
        x[1] = -1.5
        if dtype != F16:
            x[2] *= 1e-37  # the least step counts
            x[3] *= 1e-42 if dtype == F32 else 1e-38
        q, scale = ldn.quantize_rows(x)
        want_q, want_scale = oracle.quantise(x)
        assert q.dtype == torch.int8 and q.stride(0) % 16 == 0
        assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu().float(), want_q)


@pytest.mark.parametrize("C", [1, 64, 96, 1001, 5120, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_the_norm_as_integers(C, dtype):
    x, (w, b) = _rows(9, C, dtype, C), _params(C, F32, 1)
    q, scale = ldn.layer_norm_quantized(x, w, b, 1e-5)
    want, _, _, _, bound = oracle.norm(x, w, b, 1e-5)
    step = want.abs().amax(1, keepdim=True) / 127
    off = bound.amax(1, keepdim=True)
    assert ((scale.double().unsqueeze(1) - step).abs() <= off / 127 + 2 * oracle.EPS32 * step).all()
    # half a step, and what the row itself may be off; 127 steps of a scale that is off by 2 roundings
    assert ((q.double() * scale.double().unsqueeze(1) - want).abs() <= 0.5 * step + 2 * off + 127 * 4 * oracle.EPS32 * step).all()
    assert (q.abs().amax(1) == 127).all() or C == 1


def _weight(N, K, seed):
    w = torch.randn(N, K, **_gen(seed))
    return ldn.quantize_rows(w)


# one token; around the smallest tiles; around a tile of each kind; odd everything; lengths below 16 bytes; the longest sums
SHAPES = [(1, 1, 1), (1, 5120, 5120), (1, 10, 512), (2, 33, 15), (3, 128, 128), (8, 257, 1000), (9, 96, 272), (16, 512, 5119), (17, 130, 127),
          (33, 1000, 784), (64, 512, 5120), (100, 10, 5120), (129, 129, 129), (200, 777, 1001), (257, 384, 640), (300, 2049, 333),
          (512, 512, 2048), (1000, 5120, 160), (5, 40, 131071), (3000, 1100, 333), (4000, 2700, 200)]


@pytest.mark.parametrize("M, N, K", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_product(M, N, K, dtype):
    x, weight = _rows(M, K, dtype, M + N), _weight(N, K, K)
    q, scale = oracle.quantise(x)
    q, scale = q.cuda(), scale.cuda()
    bias = torch.randn(N, **_gen(3))
    for b, act in [(None, "none"), (bias, "relu"), (bias, "tanh")]:
        want, bound = oracle.product(q, scale, *weight, b, act)
        y = ldn.int8_linear(x, weight, b, activation=act)
        assert y.shape == (M, N) and y.dtype == dtype and oracle.near(y, want, bound), act
        pair = ldn.int8_linear(ldn.quantize_rows(x), weight, b, activation=act, out_dtype=dtype)
        assert torch.equal(pair, y)


@pytest.mark.parametrize("M, N, K", [(1, 33, 48), (20, 40, 64), (130, 200, 300), (300, 300, 512)])
def test_product_of_extreme_integers(M, N, K):
    f = _gen(1)
    q = torch.where(torch.rand(M, K, **f) < 0.5, -128, 127).to(torch.int8)
    w = torch.where(torch.rand(N, K, **f) < 0.5, -128, 127).to(torch.int8)
    q[0], w[0], w[-1] = -128, -128, 127
    one = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    y = ldn.int8_linear((q, one[0]), (w, one[1]))
    assert torch.equal(y.double(), q.double() @ w.double().t())  # sums below 2^24 are numbers of 32 bits


def test_product_of_the_longest_sums():
    q = torch.full((3, 131071), -128, dtype=torch.int8, device="cuda")
    y = ldn.int8_linear((q, torch.ones(3, device="cuda")), (q, torch.ones(3, device="cuda")))
    assert (y == 131071.0 * 16384).all()


@pytest.mark.parametrize("K", [48, 50])
@pytest.mark.parametrize("M", [1, 7, 40, 300])
def test_product_layouts(M, K):
    """Contiguous rows of any length, slices of wider ones, columns, a weight that starts anywhere, more than two dimensions."""
    f = _gen(M + K)
    q, w = (torch.randint(-127, 128, (n, K), dtype=torch.int8, **f) for n in (M, 30))
    sq, sw = torch.rand(M, **f), torch.rand(30, **f)
    want = ldn.int8_linear((q, sq), (w, sw))
    exact, bound = oracle.product(q, sq, w, sw, None, "none")
    assert oracle.near(want, exact, bound)

    def wider(t, before, after):
        return torch.nn.functional.pad(t, (before, after))[:, before:before + K]
    for a in (wider(q, 0, 16), wider(q, 3, 5), q.t().contiguous().t()):
        for b in (wider(w, 0, 16), wider(w, 1, 0), w.t().contiguous().t()):
            assert torch.equal(ldn.int8_linear((a, sq), (b, sw)), want)
    if M % 5 == 0:
        y = ldn.int8_linear((q.view(5, M // 5, K), sq.view(5, M // 5)), (w, sw))
        assert y.shape == (5, M // 5, 30) and torch.equal(y.view(M, 30), want)
    x = torch.randn(M, 2 * K, **f)
    assert torch.equal(ldn.int8_linear(x[:, K:], (w, sw)), ldn.int8_linear(x[:, K:].contiguous(), (w, sw)))
    assert ldn.int8_linear(x[:0, :K], (w, sw)).shape == (0, 30)
    assert torch.equal(ldn.int8_linear(x[0, :K], (w, sw)), ldn.int8_linear(x[:1, :K], (w, sw))[0])


@pytest.mark.parametrize("M", [1, 6, 40, 200])
def test_rows_that_are_not_finite_stay_by_themselves(M):
    x, weight = _rows(M + 2, 300, F32, M), _weight(50, 300, 2)
    good = ldn.int8_linear(x, weight)
    x[0, 7], x[-1, 299] = float("nan"), float("-inf")
    y = ldn.int8_linear(x, weight, activation="relu")
    assert y[0].isnan().all() and y[-1].isnan().all() and torch.equal(y[1:-1], good[1:-1].relu())


def test_a_block_as_it_answers_is_what_its_parts_are():
    x, (w, b) = _rows(70, 640, BF16, 1), _params(640, BF16, 2)
    up, down, bias = _weight(256, 640, 3), _weight(640, 256, 4), torch.randn(256, **_gen(5))
    q, scale = ldn.layer_norm_quantized(x, w, b)
    u = ldn.int8_linear((q, scale), up, bias, activation="relu", out_dtype=BF16)
    want, bound = oracle.product(q, scale, *up, bias, "relu")
    assert oracle.near(u, want, bound)
    y = ldn.int8_linear(u, down)
    uq, us = oracle.quantise(u)
    assert oracle.near(y, *oracle.product(uq.cuda(), us.cuda(), *down, None, "none"))


# ---- sizes beyond 32 bits, streams, graphs ------------------------------------------------------------------------------------------
def test_offsets_beyond_32_bits():
    C = 16384
    rows = (1 << 31) // C + 5
    x = torch.zeros(rows, C, device="cuda", dtype=F16)
    x[-3:] = _rows(3, C, F16, 1)
    w, b = _params(C, F32, 2)
    y = ldn.layer_norm(x, w, b)
    assert torch.equal(y[-3:], ldn.layer_norm(x[-3:], w, b))
    out_of = 4
    out = ldn.dropout(x, 0.25, 3, out_of)
    first = (rows - 3) * C
    kept = torch.from_numpy(oracle.words(3 * C, 3, out_of, first=first) >= np.uint64(1 << 30)).view(3, C)
    assert torch.equal(out[-3:], oracle.dropped(x[-3:], kept, 0.25).to(F16))
    del y
    weight = _weight(16, C, 5)
    y = ldn.int8_linear(x, weight)
    assert torch.equal(y[-3:], ldn.int8_linear(x[-3:].clone(), weight))
    h = ldn.dropout_add_layer_norm(out, x, w, b, 0.25, 3, out_of)[1]
    assert torch.equal(h[-3:], (x[-3:].float() + oracle.dropped(out[-3:], kept, 0.25)).to(F16))


def test_gradients_beyond_32_bits():
    C = 16384
    rows = (1 << 31) // C + 3
    x = torch.zeros(rows, C, device="cuda", dtype=F16)
    x[-2:] = _rows(2, C, F16, 1)
    w = _params(C, F32, 2)[0].requires_grad_()
    g = torch.zeros(rows, C, device="cuda", dtype=F16)
    g[-2:] = torch.randn(2, C, **_gen(3)).half()
    x.requires_grad_()
    gx, gw = torch.autograd.grad(ldn.layer_norm(x, w, None), (x, w), g)
    small = x.detach()[-2:].clone().requires_grad_()
    sx, sw = torch.autograd.grad(ldn.layer_norm(small, w, None), (small, w), g[-2:])
    assert torch.equal(gx[-2:], sx) and torch.allclose(gw, sw, rtol=1e-5, atol=1e-6) and not gx[:4].any()


def _everything(x, r, w, b, g, weight, seed):
    y, h = ldn.dropout_add_layer_norm(x, r, w, b, 0.1, seed)
    n = ldn.layer_norm(h, w, b)
    d = ldn.dropout(n, 0.2, seed, 5)
    grads = torch.autograd.grad((y, d), (x, r, w, b), (g, g))
    with torch.no_grad():
        return (y, h, n, d) + grads + (ldn.int8_linear(x, weight), ldn.int8_linear(ldn.layer_norm_quantized(x, w, b), weight))


def _case():
    x, r = (_rows(150, 1000, F32, k).requires_grad_() for k in (1, 2))
    w, b = (t.requires_grad_() for t in _params(1000, F32, 3))
    return x, r, w, b, torch.randn(150, 1000, **_gen(4)), _weight(200, 1000, 5)


def test_another_stream():
    case = _case()
    want = _everything(*case, 11)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    late = [t.detach().clone().zero_().requires_grad_(t.requires_grad) for t in case[:5]]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        with torch.no_grad():
            for a, t in zip(late, case):
                a.copy_(t)
        got = _everything(*late, case[5], 11)
    stream.synchronize()
    assert all(torch.equal(a, t) for a, t in zip(got, want))


def test_recorded_in_a_graph():
    case = _case()
    state = torch.tensor([11, 0], device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _everything(*case, state)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = _everything(*case, state)
    for offset in (0, 3):
        state[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        eager = _everything(*case, torch.tensor([11, offset], device="cuda"))
        assert all(torch.equal(a, t) for a, t in zip(got, eager))


# ---- what is refused ------------------------------------------------------------------------------------------------------------------
def test_refusals():
    x, (w, b), weight = _rows(4, 8, F32, 1), _params(8, F32, 2), _weight(3, 8, 3)
    q, s = ldn.quantize_rows(x)
    refused = [
        lambda: ldn.layer_norm(x.double(), w, b), lambda: ldn.layer_norm(x, w[:7], b), lambda: ldn.layer_norm(x, w.half(), b.half()),
        lambda: ldn.layer_norm(x, w, b.double()), lambda: ldn.layer_norm(x.half(), w, b.half()), lambda: ldn.layer_norm(x, w.cpu(), b),
        lambda: ldn.layer_norm(x, w, b, -1.0), lambda: ldn.layer_norm(x[0, 0], w, b), lambda: ldn.layer_norm(x[:, :0], None, None),
        lambda: ldn.dropout(x, 1.1, 1), lambda: ldn.dropout(x, float("nan"), 1), lambda: ldn.dropout(x.int(), 0.1, 1),
        lambda: ldn.dropout(x, 0.1, torch.zeros(3, dtype=torch.int64, device="cuda")), lambda: ldn.dropout(x, 0.1, torch.zeros(2)),
        lambda: ldn.dropout(x, 0.1, 1, residual=x[:2]), lambda: ldn.dropout(x, 0.1, 1, residual=x.half()),
        lambda: ldn.dropout_add_layer_norm(x, x[:1], w, b, 0.1, 1), lambda: ldn.dropout_add_layer_norm(x, x, w, b, -0.1, 1),
        lambda: ldn.quantize_rows(x.double()), lambda: ldn.quantize_rows(x.clone().requires_grad_()),
        lambda: ldn.layer_norm_quantized(x, w.clone().requires_grad_(), b), lambda: ldn.int8_linear(x[:, :7], weight),
        lambda: ldn.int8_linear(x, (weight[0].float(), weight[1])), lambda: ldn.int8_linear(x, (weight[0], weight[1][:2])),
        lambda: ldn.int8_linear(x, weight, b), lambda: ldn.int8_linear((q, s[:3]), weight), lambda: ldn.int8_linear((x, s), weight),
        lambda: ldn.int8_linear(x, weight, out_dtype=torch.float64), lambda: ldn.int8_linear(x.clone().requires_grad_(), weight),
        lambda: ldn.int8_linear((q[:1].expand(4, 8), s), weight),
        lambda: torch.vmap(lambda t: ldn.layer_norm(t, w, b))(torch.randn(2, 4, 8, device="cuda")),
    ]
    before = lib.ldn_kernel_launches()
    for call in refused:
        with pytest.raises(RuntimeError):
            call()
    assert lib.ldn_kernel_launches() == before
    with pytest.raises(RuntimeError, match="differentiated again"):
        z = x.clone().requires_grad_()
        g, = torch.autograd.grad(ldn.layer_norm(z, w, b), z, torch.ones_like(x).requires_grad_(), create_graph=True)
    torch.cuda.synchronize()


def test_layers_train_and_answer():
    torch.manual_seed(0)
    norm, drop, linear = ldn.LayerNorm(96).cuda(), ldn.Dropout(0.5, seed=3), torch.nn.Linear(96, 20).cuda()
    x = _rows(32, 96, F32, 1)
    first, second = drop(x), drop(x)
    assert not torch.equal(first, second)
    y = linear(norm(drop(x, x)))
    y.sum().backward()
    assert norm.weight.grad.shape == (96,) and linear.weight.grad is not None
    small = ldn.Int8Linear.from_linear(linear)
    with torch.no_grad():
        n = norm.eval()(x)
        want = linear(n)
        # a row's and an output's steps are their largest values over 127: half a step each on 96 terms, at random
        off = 6 * (96 ** 0.5) * (n.abs().amax() / 254 * linear.weight.abs().amax() * 2)
        assert (small(n) - want).abs().max() <= off
    again = ldn.Int8Linear(torch.zeros(20, 96, device="cuda"), torch.zeros(20, device="cuda"))
    again.load_state_dict(small.state_dict())
    assert torch.equal(again(n), small(n))


# ---- the head as it is used -----------------------------------------------------------------------------------------------------------
def _model(**kwargs):
    torch.manual_seed(0)
    model = ldn.ResidualModel(4, 96, [1, 8, 8], hidden=128, blocks=3, seed=11, **kwargs).cuda()
    ldn.set_p_norm(model, float("inf"))
    return model


def test_a_head_is_its_formula():
    model = _model(dropout=0.2)
    head, features = model.head, _rows(50, 96, F32, 1).requires_grad_()
    got = head(features)

    def plain(h):
        h = h.double()
        y = oracle.norm(h, head.norm[0].weight, head.norm[0].bias, 1e-5)[0]
        for i in range(3):
            u = torch.relu(y @ head.up[i].weight.double().t() + head.up[i].bias.double()) @ head.down[i].weight.double().t() + head.down[i].bias.double()
            h = h + torch.where(oracle.keep((50, 96), 0.2, 11 + i, 0).cuda(), u / 0.8, 0.0)
            y = oracle.norm(h, head.norm[i + 1].weight, head.norm[i + 1].bias, 1e-5)[0]
        return y @ head.final.weight.double().t() + head.final.bias.double()
    want = plain(features)
    # four products of up to 128 terms, three blocks: some hundred roundings of numbers of the stream's size
    assert (got - want).abs().max() <= 1000 * oracle.EPS32 * want.abs().max()
    v = torch.randn(50, 10, **_gen(2))
    params = [p for p in head.parameters()]
    for a, b in zip(torch.autograd.grad(got, [features] + params, v), torch.autograd.grad((want * v).sum(), [features] + params)):
        assert (a - b).abs().max() <= 4000 * oracle.EPS32 * b.abs().max()


def test_a_model_learns_and_answers():
    model = _model()
    x = torch.rand(64, 1, 8, 8, **_gen(1))
    targets = torch.arange(64, device="cuda") % 10
    from l_inf_dist_net_v2_b200.optim import FusedAdam
    optimizer = FusedAdam(model.parameters(), lr=1e-3)
    losses = []
    for _ in range(40):
        loss = torch.nn.functional.cross_entropy(model(x), targets)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    assert losses[-1] < 0.5 * losses[0]
    with torch.no_grad():
        want = model.eval()(x)
        assert torch.equal(model(x), want)  # no dropout
        got = model.quantize()(x)
        assert (got - want).abs().max() <= 0.1 * want.abs().max() and (got.argmax(1) == want.argmax(1)).float().mean() >= 0.9
        assert torch.equal(model(x[:1]), got[:1]) and torch.equal(model(x[:30]), got[:30])  # whatever the kernel for the batch
    assert not torch.equal(model.train()(x), want)
    again = _model()
    again.load_state_dict(model.state_dict())
    with torch.no_grad():
        assert torch.equal(again.eval()(x), model.eval()(x))


def test_a_training_step_in_a_graph_draws_again():
    """Masks of a replay follow the words on the device, gradients those of the same replay."""
    x, r = (_rows(20, 64, F32, k).requires_grad_() for k in (1, 2))
    w, b = (t.requires_grad_() for t in _params(64, F32, 3))
    g = torch.randn(20, 64, **_gen(4))
    state = torch.tensor([5, 0], device="cuda")

    def step():
        y, h = ldn.dropout_add_layer_norm(x, r, w, b, 0.5, state)
        grads = torch.autograd.grad((y, h), (x, r), (g, g))
        state[1] += 1
        return h, grads[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        h, gx = step()
    for offset in (1, 2, 3):
        graph.replay()
        torch.cuda.synchronize()
        kept = oracle.keep((20, 64), 0.5, 5, offset).cuda()
        assert torch.equal(h, r + oracle.dropped(x, kept, 0.5)) and not gx[~kept].any()
