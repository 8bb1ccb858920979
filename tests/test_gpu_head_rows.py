"""The head's row kernels with several rows per thread, at values where statistics are extreme, and results of very many outputs."""
import pytest
import torch

import head_oracle as oracle
import l_inf_dist_net_v2_b200 as ldn
from l_inf_dist_net_v2_b200._lib import lib

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAMES = {F32: 0, F16: 1, BF16: 2}


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _params(C, dtype, seed):
    f = _gen(seed)
    return (1 + 0.3 * torch.randn(C, **f)).to(dtype), (0.3 * torch.randn(C, **f)).to(dtype)


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
