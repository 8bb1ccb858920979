"""The head's layers and models in the ways that a program uses them: differentiated again, recomputed, in mixed precision, moved,
answering in integers while their weights change, from several threads."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import l_inf_dist_net_v2_b200 as ldn

pytestmark = pytest.mark.gpu


def _gen(seed):
    return dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _model(**kwargs):
    torch.manual_seed(0)
    model = ldn.ResidualModel(4, 96, [1, 8, 8], hidden=120, blocks=3, seed=11, **kwargs).cuda()
    ldn.set_p_norm(model, float("inf"))
    return model


# ---- recomputed ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_head_has_the_gradients_of_its_masks(reentrant):
    a = _model(dropout=0.4).head
    b = copy.deepcopy(a)
    xs = [torch.randn(30, 96, **_gen(k)).requires_grad_() for k in range(2)]
    outs, wants = [checkpoint(a, x, use_reentrant=reentrant) for x in xs], [b(x) for x in xs]
    for out, want, x in zip(outs, wants, xs):
        assert torch.equal(out, want)
        out.square().sum().backward()
        g, x.grad = x.grad, None
        want.square().sum().backward()
        assert torch.equal(x.grad, g)
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(a.parameters(), b.parameters()))
