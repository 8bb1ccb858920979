"""The head's row kernels with several rows per thread, at values where statistics are extreme, and results of very many outputs."""
import pytest
import torch

import l_inf_dist_net_v2_b200 as ldn

pytestmark = pytest.mark.gpu


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


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
