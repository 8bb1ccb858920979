"""The head's row kernels with several rows per thread, at values where statistics are extreme, and results of very many outputs."""
import pytest
import torch

import head_oracle as oracle
import l_inf_dist_net_v2_b200 as ldn
from l_inf_dist_net_v2_b200._lib import lib

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAMES = {F32: 0, F16: 1, BF16: 2}
MANY = [147, 149, 1000, 5000]
WIDTHS = [(96, BF16), (512, F32), (1001, F16), (5120, BF16)]


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _rows(rows, C, dtype, seed, pitch=None):
    f = _gen(seed)
    x = torch.randn(rows, pitch or C, **f) * (torch.rand(rows, 1, **f) * 2 + 0.5) + torch.randn(rows, 1, **f)
    return x.to(dtype)[:, :C]


def _params(C, dtype, seed):
    f = _gen(seed)
    return (1 + 0.3 * torch.randn(C, **f)).to(dtype), (0.3 * torch.randn(C, **f)).to(dtype)


# ---- several rows per thread --------------------------------------------------------------------------------------------------------
def _joined(rows, C, dtype, pitch=None):
    p, seed, offset = 0.3, 98765432109, 5
    x, r = (_rows(rows, C, dtype, rows + k, pitch).detach().requires_grad_() for k in (0, 1))
    w, b = (t.requires_grad_() for t in _params(C, F32, 1))
    kept = oracle.keep((rows, C), p, seed, offset).cuda()
    y, h = ldn.dropout_add_layer_norm(x, r, w, b, p, seed, offset)
    want_h = (r.detach().float() + oracle.dropped(x.detach(), kept, p)).to(dtype)
    assert torch.equal(h, want_h)
    want, _, _, _, bound = oracle.norm(want_h, w.detach(), b.detach(), 1e-5)
    assert oracle.near(y.detach(), want, bound)
    gy, gh = (torch.randn(rows, C, **_gen(k)).to(dtype) for k in (2, 3))
    got = torch.autograd.grad((y, h), (x, r, w, b), (gy, gh), retain_graph=True)
    (want_x, off_x), sums_w, sums_b = oracle.norm_grad(gy, want_h, w.detach(), 1e-5)
    whole = want_x + gh.double()
    off = off_x + oracle.EPS32 * whole.abs()
    scale = 1 / (1 - p)
    assert oracle.near(got[0], torch.where(kept, whole * scale, 0.0), off * scale + 4 * oracle.EPS32 * whole.abs())
    assert oracle.near(got[1], whole, off)
    assert oracle.near(got[2], *sums_w) and oracle.near(got[3], *sums_b)
    again = torch.autograd.grad((y, h), (x, r, w, b), (gy, gh))
    assert all(torch.equal(s, t) for s, t in zip(got, again))  # sums in a fixed order


@pytest.mark.parametrize("rows", MANY)
@pytest.mark.parametrize("C, dtype", WIDTHS)
def test_joined_over_many_rows(rows, C, dtype):
    _joined(rows, C, dtype)


@pytest.mark.parametrize("rows", MANY)
@pytest.mark.parametrize("C, dtype", WIDTHS)
def test_integers_over_many_rows(rows, C, dtype):
    x, (w, b) = _rows(rows, C, dtype, rows), _params(C, F32, 1)
    q, scale = ldn.quantize_rows(x)
    want_q, want_scale = oracle.quantise(x)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu().float(), want_q)
    _normed_integers(x, w, b)


def _normed_integers(x, w, b):
    q, scale = ldn.layer_norm_quantized(x, w, b, 1e-5)
    want, _, _, _, bound = oracle.norm(x, w, b, 1e-5)
    step = want.abs().amax(1, keepdim=True) / 127
    off = bound.amax(1, keepdim=True)
    assert ((scale.double().unsqueeze(1) - step).abs() <= off / 127 + 2 * oracle.EPS32 * step).all()
    # half a step, and what the row itself may be off; 127 steps of a scale that is off by 2 roundings
    assert ((q.double() * scale.double().unsqueeze(1) - want).abs() <= 0.5 * step + 2 * off + 127 * 4 * oracle.EPS32 * step).all()


@pytest.mark.parametrize("rows", [5, 5000])
@pytest.mark.parametrize("C, pitch, dtype", [(96, 104, BF16), (96, 100, F32), (5120, 5128, F16)])
def test_slices_whose_rows_start_at_multiples_of_16_bytes(rows, C, pitch, dtype):
    _joined(rows, C, dtype, pitch)
    x, (w, b) = _rows(rows, C, dtype, 3, pitch), _params(C, F32, 1)
    _normed_integers(x, w, b)
    whole = x.contiguous()
    assert all(torch.equal(s, t) for s, t in zip(ldn.quantize_rows(x), ldn.quantize_rows(whole)))
    assert torch.equal(ldn.layer_norm(x, w, b), ldn.layer_norm(whole, w, b))
    grads = []
    g = torch.randn(rows, C, **_gen(4)).to(dtype)
    for t in (x, whole):
        t = t.detach().requires_grad_()
        u, v = (s.detach().requires_grad_() for s in (w, b))
        grads.append(torch.autograd.grad(ldn.layer_norm(t, u, v), (t, u, v), g))
    assert all(torch.equal(s, t) for s, t in zip(*grads))


def test_a_block_repeats_itself():
    """The same integers and the same bits every time, with other calls in between, and integers as near to 64 bits as 32 allow."""
    x, (w, b) = _rows(512, 5120, BF16, 1), _params(5120, BF16, 2)
    up, down = ldn.quantize_rows(torch.randn(2048, 5120, **_gen(3))), ldn.quantize_rows(torch.randn(5120, 2048, **_gen(4)))
    bias = torch.randn(2048, **_gen(5))

    def block(rows):
        q = ldn.layer_norm_quantized(rows, w, b)
        u = ldn.int8_linear(q, up, bias, activation="relu", out_dtype=BF16)
        return q + (u, ldn.int8_linear(u, down))
    first = block(x)
    other = _rows(300, 5120, BF16, 6)
    for _ in range(20):
        block(other)
        assert all(torch.equal(s, t) for s, t in zip(block(x), first))


# ---- statistics at the ends of their range --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", [2, 10, 96, 100, 1000, 1001, 4096, 5000, 5120, 16000])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("joined", [False, True])
def test_gradients_of_rows_whose_mean_is_many_deviations_away(C, dtype, joined):
    """Rows of one value: x - mean is 0 and the gradient rstd (a - mean(a)), whatever mean * rstd is."""
    rows, value, rstd = 300, 2.0 ** 110, 2.0 ** 20
    x = torch.full((rows, C), value, device="cuda", dtype=dtype)
    g, (w, _) = torch.randn(rows, C, **_gen(C)).to(dtype), _params(C, F32, 1)
    stats = torch.tensor([value, rstd], device="cuda").repeat_interleave(rows)
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    mean_at, rstd_at = stats.data_ptr(), stats.data_ptr() + 4 * rows
    stream = torch.cuda.current_stream().cuda_stream
    if joined:
        status = lib.ldn_dropout_add_layer_norm_backward(g.data_ptr(), None, x.data_ptr(), rows, C, NAMES[dtype], mean_at, rstd_at,
                                                         w.data_ptr(), 0, 0.0, 1, 0, None, gx.data_ptr(), None, gw.data_ptr(),
                                                         gb.data_ptr(), stream)
    else:
        status = lib.ldn_layer_norm_backward(g.data_ptr(), x.data_ptr(), C, rows, C, NAMES[dtype], mean_at, rstd_at, w.data_ptr(), 0,
                                             gx.data_ptr(), gw.data_ptr(), gb.data_ptr(), stream)
    assert status == 0
    a = g.double() * w.double()
    # a chain of at most C / 128 + 48 additions, as in the oracle
    off = rstd * (C / 128 + 48) * oracle.EPS32 * 2 * (a.abs() + a.abs().mean(1, keepdim=True))
    assert oracle.near(gx, rstd * (a - a.mean(1, keepdim=True)), off)
    assert not gw.any()
    assert oracle.near(gb, g.double().sum(0), (rows / 4 + 64) * oracle.EPS32 * g.double().abs().sum(0))


# ---- very many outputs ------------------------------------------------------------------------------------------------------------------
def test_sixteen_tokens_of_eighty_million_outputs():
    """Rows of 320 MB: sixteen of them are more than 32 bits count."""
    N, K, M = 80_000_000, 16, 16
    w = torch.randint(-127, 128, (N, K), dtype=torch.int8, **_gen(1))
    weight = (w, torch.rand(N, **_gen(2)))
    x = ldn.quantize_rows(torch.randn(M, K, **_gen(3)))
    y = ldn.int8_linear(x, weight)
    for m in range(M):
        assert torch.equal(y[m], ldn.int8_linear((x[0][m], x[1][m]), weight)), m
