"""Distillation from a teacher's top logits on a B200 against the formulas in 64 bits."""
import math

import pytest
import torch

import distil_oracle as oracle
import head_oracle
import l_inf_dist_net_v2_b200 as ldn

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def made(rows, V, k, dtype, teacher=None, ragged=False, masked=False, layout="plain", seed=0):
    f = dict(device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + V))
    x = 2 * torch.randn(rows, V, **f) + 3 * torch.randn(rows, 1, **f)
    t = 0.5 * x + torch.randn(rows, V, **f)
    if masked:
        gone = torch.rand(rows, V, **f) < 0.2
        gone[:, :k] = False
        x.masked_fill_(gone, -math.inf)
        t.masked_fill_(gone, -math.inf)
    values, indices = t.topk(k, 1)
    targets = indices[:, -1].clone()
    if ragged:
        indices = torch.where(torch.rand(rows, k, **f) < torch.rand(rows, 1, **f), indices, -1)
        indices[0] = -1
        targets[1::3] = -1
    x = x.to(dtype)
    if layout == "slice":
        x = torch.nn.functional.pad(x, (0, 3))[:, :V]
    if layout == "shifted":
        flat = torch.empty(rows * V + 1, device="cuda", dtype=dtype)
        flat[1:] = x.reshape(-1)
        x = flat[1:].view(rows, V)
    return x, values.to(teacher or dtype), indices, targets, torch.randn(rows, **f)


def check(x, values, indices, targets, up, tau, mix):
    leaf = x.detach().requires_grad_()
    losses = ldn.distillation_loss(leaf, values, indices, targets, tau, mix, "none")
    want, bound, dx, off = oracle.loss_and_gradient(x, values, indices, targets, tau, mix, up)
    assert losses.dtype == torch.float32 and losses.shape == x.shape[:-1]
    assert head_oracle.near(losses.detach(), want, bound)
    got, = torch.autograd.grad(losses, leaf, up)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert head_oracle.near(got, dx, off)
    with torch.no_grad():
        assert torch.equal(ldn.distillation_loss(x, values, indices, targets, tau, mix, "none"), losses)
    for reduction, by in (("sum", 1.0), ("mean", 1.0 / x.size(0))):
        leaf = x.detach().requires_grad_()
        loss = ldn.distillation_loss(leaf, values, indices, targets, tau, mix, reduction)
        # (a chain of rows / 4096 + 24 additions)
        near = (bound.sum() + (x.size(0) / 4096 + 28) * head_oracle.EPS32 * want.abs().sum()) * by
        assert loss.dim() == 0 and head_oracle.near(loss.detach(), want.sum() * by, near)
        same, = torch.autograd.grad(loss, leaf, torch.full_like(loss, 3.0))
        _, _, dx1, off1 = oracle.loss_and_gradient(x, values, indices, targets, tau, mix, torch.full_like(up, 3.0 * by))
        assert head_oracle.near(same, dx1, off1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, V, k", [(1, 1, 1), (5, 2, 2), (33, 10, 3), (9, 33, 33), (7, 1000, 20), (3, 2048, 64), (3, 2049, 64), (2, 4097, 1),
                                        (5, 40001, 100), (1, 131072, 1000), (300, 8192, 7), (2, 16384, 3), (3000, 17, 2)])
def test_sizes(rows, V, k, dtype):
    for tau, mix in ((1.0, 0.0), (2.0, 0.3), (1.0, 0.4), (4.0, 1.0)):
        check(*made(rows, V, k, dtype), tau, mix)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [10, 1001, 5003])
def test_lists_of_different_lengths_masks_and_layouts(V, dtype):
    for layout in ("plain", "slice", "shifted"):
        check(*made(13, V, 5, dtype, ragged=True, masked=True, layout=layout), 2.0, 0.3)
        check(*made(13, V, 5, dtype, teacher=F32, ragged=True, layout=layout), 0.5, 0.0)


@pytest.mark.parametrize("V", [10, 1001, 5003])
def test_one_class_several_times_and_in_any_order(V):
    for dtype in TYPES:
        x, values, indices, targets, up = made(6, V, 5, dtype)
        indices[:, 3] = indices[:, 0]
        indices[1] = indices[1, 0]
        targets[2] = indices[2, 3]
        check(x, values.flip(1), indices, targets, up, 2.0, 0.3)


@pytest.mark.parametrize("V", [12, 3000])
def test_rows_that_say_nothing_and_rows_that_are_wrong(V):
    x, values, indices, targets, up = made(8, V, 4, F32)
    x[0] = -math.inf            # no choice, no list, no label
    indices[0], targets[0] = -1, -1
    values[1] = -math.inf       # a list of nothing but minus infinity
    targets[1] = -1
    indices[2, 1] = V           # beyond the classes
    targets[3] = V
    x[4, 5] = math.nan
    x[5, 5] = math.inf
    values[6, 0] = math.nan
    x[7, indices[7, 0]] = -math.inf  # what the teacher prefers is no choice
    leaf = x.detach().requires_grad_()
    losses = ldn.distillation_loss(leaf, values, indices, targets, 2.0, 0.3, "none")
    dx, = torch.autograd.grad(losses.sum(), leaf)
    assert torch.equal(losses[:2].detach(), torch.zeros(2, device="cuda")) and torch.equal(dx[:2], torch.zeros_like(dx[:2]))
    assert losses[2:7].isnan().all() and dx[2:6].isnan().all() and dx[6, indices[6]].isnan().all()
    assert losses[7] == math.inf and dx[7].isfinite().all()


def test_shapes_and_no_rows():
    x, values, indices, targets, up = made(12, 50, 4, F32)
    want = ldn.distillation_loss(x, values, indices, targets, 2.0, 0.3, "none")
    cube = ldn.distillation_loss(x.view(3, 4, 50), values.view(3, 4, 4), indices.view(3, 4, 4), targets.view(3, 4), 2.0, 0.3, "none")
    assert torch.equal(cube, want.view(3, 4))
    assert torch.equal(ldn.distillation_loss(x[0], values[0], indices[0], targets[0], 2.0, 0.3, "none"), want[0])
    turned = ldn.distillation_loss(x.t().contiguous().t(), values.t().contiguous().t(), indices.t().contiguous().t(), targets, 2.0, 0.3, "none")
    assert torch.equal(turned, want)
    for dtype in TYPES:
        leaf = x[:0].to(dtype).requires_grad_()
        losses = ldn.distillation_loss(leaf, values[:0], indices[:0], reduction="none")
        assert losses.shape == (0,) and torch.autograd.grad(losses, leaf, losses.detach())[0].shape == (0, 50)
        assert ldn.distillation_loss(leaf, values[:0], indices[:0], reduction="sum") == 0


def test_a_teacher_of_all_classes_is_the_plain_loss():
    """With every class in the list it is the Kullback-Leibler divergence, and with mix = 1 the cross-entropy, of torch in 64 bits."""
    x, values, indices, targets, up = made(20, 60, 60, F32)
    q = torch.log_softmax(x.double() / 3, 1)
    p = torch.zeros_like(q).scatter_(1, indices, torch.softmax(values.double() / 3, 1))
    want = torch.nn.functional.kl_div(q, p, reduction="batchmean") * 9
    assert abs(ldn.distillation_loss(x, values, indices, temperature=3.0) - want) <= 1e-5 * want
    want = torch.nn.functional.cross_entropy(x.double(), targets)
    assert abs(ldn.distillation_loss(x, values, indices, targets, 3.0, 1.0) - want) <= 1e-5 * want


def test_gradient_against_differences():
    x, values, indices, targets, up = made(5, 40, 6, F32, ragged=True)
    leaf = x.requires_grad_()
    for tau, mix in ((1.0, 0.0), (2.0, 0.4)):
        g, = torch.autograd.grad(ldn.distillation_loss(leaf, values, indices, targets, tau, mix, "none"), leaf, up)
        step = torch.randn_like(x)
        a, b = ((oracle.loss_and_gradient(x.detach().double() + s * 2 ** -10 * step, values, indices, targets, tau, mix, up)[0] * up.double()).sum()
                for s in (1, -1))
        assert abs((a - b) / 2 ** -9 - (g.double() * step).sum()) <= 2.0 ** -16 * (up.abs().sum() + (g * step).abs().sum())


def test_differentiated_twice_says_so():
    x, values, indices, targets, up = made(5, 40, 6, F32)
    leaf = x.requires_grad_()
    g, = torch.autograd.grad(ldn.distillation_loss(leaf, values, indices), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        g.square().sum().backward()


def test_offsets_beyond_32_bits():
    rows, V = 20000, 131072
    x = torch.empty(rows, V, device="cuda", dtype=BF16).normal_()
    values, indices = x[:, :5].clone(), torch.randint(V, (rows, 5), device="cuda")
    targets, up = indices[:, 0].clone(), torch.zeros(rows, device="cuda")
    up[-3:] = 1.0
    leaf = x.requires_grad_()
    losses = ldn.distillation_loss(leaf, values, indices, targets, 2.0, 0.3, "none")
    dx, = torch.autograd.grad(losses, leaf, up)
    want, bound, grad, off = oracle.loss_and_gradient(x.detach()[-3:], values[-3:], indices[-3:], targets[-3:], 2.0, 0.3, up[-3:])
    assert head_oracle.near(losses.detach()[-3:], want, bound) and head_oracle.near(dx[-3:], grad, off) and not dx[:-3].any()


def test_refusals():
    x, values, indices, targets, _ = made(4, 9, 3, F32)
    loss = ldn.distillation_loss
    refused = [
        lambda: loss(x.double(), values, indices), lambda: loss(x, values.double(), indices), lambda: loss(x, values, indices.int()),
        lambda: loss(x, values[:3], indices[:3]), lambda: loss(x, values, indices[:, :2]), lambda: loss(x, values[:, :0], indices[:, :0]),
        lambda: loss(x, values.cpu(), indices), lambda: loss(x, values, indices, targets[:3], mix=0.5), lambda: loss(x, values, indices, targets.int(), mix=0.5),
        lambda: loss(x, values, indices, targets.float(), mix=0.5), lambda: loss(x, values, indices, temperature=0.0),
        lambda: loss(x, values, indices, temperature=-1.0), lambda: loss(x, values, indices, temperature=math.inf),
        lambda: loss(x, values, indices, temperature=math.nan), lambda: loss(x, values, indices, targets, mix=1.5),
        lambda: loss(x, values, indices, targets, mix=-0.5), lambda: loss(x, values.requires_grad_(), indices), lambda: loss(x[:, :0], values, indices),
        lambda: loss(x, torch.zeros(4, 1025, device="cuda"), torch.zeros(4, 1025, device="cuda", dtype=torch.int64)),
        lambda: torch.vmap(lambda a: loss(a, values.detach(), indices))(x[None]),
    ]
    before = ldn._lib.lib.ldn_kernel_launches()
    for attempt in refused:
        with pytest.raises(RuntimeError):
            attempt()
    assert ldn._lib.lib.ldn_kernel_launches() == before


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, V, k", [(600, 8193, 5), (1000, 3001, 128), (777, 10007, 129), (4000, 8200, 33), (650, 33000, 1)])
def test_many_long_rows(rows, V, k, dtype):
    check(*made(rows, V, k, dtype, ragged=True), 1.0, 0.3)
    check(*made(rows, V, k, dtype, layout="slice"), 2.0, 0.0)
    x, values, indices, targets, up = made(rows, V, k, dtype, masked=True, layout="shifted")
    x[1], x[2, V // 2:], x[rows - 1, :V - 1] = -math.inf, -math.inf, -math.inf
    x[3, 0], x[4, V - 1], x[5, 17] = math.nan, math.inf, math.nan
    indices[1], targets[1] = -1, -1
    indices[2], targets[2] = torch.arange(k, device="cuda"), 1
    indices[rows - 1], targets[rows - 1] = -1, V - 1
    indices[rows - 1, 0] = V - 1
    losses = ldn.distillation_loss(x, values, indices, targets, 2.0, 0.3, "none")
    assert losses[3:6].isnan().all() and losses[1] == 0
    keep = [0, 2] + list(range(6, rows))
    want, bound, _, _ = oracle.loss_and_gradient(x[keep], values[keep], indices[keep], targets[keep], 2.0, 0.3, up[keep])
    # (the last row's only class may be one that is no choice: a row of nothing but minus infinity with a label is not a number)
    some = torch.tensor([bool((x[i] > -math.inf).any()) for i in keep], device="cuda")
    assert torch.equal(losses[keep].isfinite(), some) and losses[keep][~some].isnan().all()
    assert head_oracle.near(losses[keep][some], want[some], bound[some])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, V", [(40, 12), (9, 1001), (6, 5003), (700, 8193), (6, 40001)])
def test_a_term_without_weight_is_none(rows, V, dtype):
    """With mix = 1 what the teacher says does not count, a class that is no choice and values that are no numbers among it."""
    x, values, indices, targets, up = made(rows, V, 4, dtype)
    x[0, indices[0, 0]] = x[2, indices[2, 1]] = -math.inf
    targets[0], targets[2] = indices[0, 1], indices[2, 0]
    values[1, 0], values[1, 1] = math.nan, math.inf
    values[3] = -math.inf
    targets[4] = -1
    for tau in (1.0, 2.0, 3.0):
        leaf = x.detach().requires_grad_()
        losses = ldn.distillation_loss(leaf, values, indices, targets, tau, 1.0, "none")
        want, bound, dx, off = oracle.loss_and_gradient(x, torch.zeros_like(values), torch.full_like(indices, -1), targets, tau, 1.0, up)
        assert want.isfinite().all() and head_oracle.near(losses.detach(), want, bound)
        assert head_oracle.near(torch.autograd.grad(losses, leaf, up)[0], dx, off)
        assert ldn.distillation_loss(x, values, indices, targets, tau, 1.0).isfinite()
    indices[5 % rows, 2] = V  # (an index beyond the classes is wrong whatever it counts)
    leaf = x.detach().requires_grad_()
    losses = ldn.distillation_loss(leaf, values, indices, targets, 2.0, 1.0, "none")
    dx, = torch.autograd.grad(losses, leaf, torch.ones_like(losses))
    assert losses[5 % rows].isnan() and dx[5 % rows].isnan().all() and losses.isnan().sum() == 1


@pytest.mark.parametrize("V", [12, 5003])
def test_labels_without_weight_are_none_in_the_library(V):
    x, values, indices, targets, up = made(6, V, 4, F32)
    x[0, targets[0]] = -math.inf
    indices[0] = torch.where(indices[0] == targets[0], -1, indices[0])
    losses, stats, grad = torch.empty(6, device="cuda"), torch.empty(5, 6, device="cuda"), torch.empty_like(x)
    lib, at = ldn._lib.lib, [t.data_ptr() for t in (x, values, indices, targets)]
    assert lib.ldn_distillation(at[0], V, 6, V, 0, at[1], 0, at[2], 4, at[3], 2.0, 1.0, 0.0, losses.data_ptr(), stats.data_ptr(), 1.0, None, None) == 0
    assert lib.ldn_distillation_backward(at[0], V, 6, V, 0, at[1], 0, at[2], 4, at[3], 2.0, 1.0, 0.0, stats.data_ptr(), up.data_ptr(), 1, 1.0,
                                         grad.data_ptr(), None) == 0
    leaf = x.detach().requires_grad_()
    want = ldn.distillation_loss(leaf, values, indices, temperature=2.0, reduction="none")
    assert want.isfinite().all() and torch.equal(losses, want.detach())
    assert torch.equal(grad, torch.autograd.grad(want, leaf, up)[0])


@pytest.mark.parametrize("V", [10, 1001, 5003])
def test_entries_of_one_class_against_their_dense_sum(V):
    """With P the sum of a class's p, made densely in 64 bits: the gradient is that of P, the loss the divergence of P and, as log p is each
    entry's own, sum p log p - sum P log P less."""
    tau, k = 2.0, 6
    x, values, indices, _, up = made(8, V, k, F32)
    indices[:, 3] = indices[:, 0]
    indices[:, 5] = indices[:, 0]
    indices[1] = indices[1, 0]
    indices[2, 4] = -1
    x[0] = -math.inf  # two equal entries of one class, which is all that there is to choose
    x[0, 7], indices[0], values[0, :2] = 0.5, torch.tensor([7, 7, -1, -1, -1, -1], device="cuda"), 1.25
    leaf = x.detach().requires_grad_()
    losses = ldn.distillation_loss(leaf, values, indices, temperature=tau, reduction="none")
    dx, = torch.autograd.grad(losses, leaf, up)
    there = indices >= 0
    p = torch.softmax(torch.where(there, values.double() / tau, -math.inf), 1)
    P = torch.zeros(8, V, device="cuda", dtype=torch.float64).scatter_add_(1, indices.clamp_min(0), torch.where(there, p, 0.0))
    log_q = torch.log_softmax(x.double() / tau, 1)
    dense = (torch.xlogy(P, P) - torch.where(P > 0, P * log_q, 0.0)).sum(1)
    want = tau ** 2 * (dense + torch.xlogy(p, p).sum(1) - torch.xlogy(P, P).sum(1))
    _, bound, _, off = oracle.loss_and_gradient(x, values, indices, None, tau, 0.0, up)
    assert head_oracle.near(losses.detach(), want, bound)
    assert head_oracle.near(dx, up.double()[:, None] * tau * (log_q.exp() - P), off)
    assert abs(losses[0] + tau ** 2 * math.log(2)) <= 2.0 ** -20 and losses[0] < 0


@pytest.mark.parametrize("rows, V", [(6, 12), (6, 5003), (700, 8193)])
def test_a_teacher_of_the_lowest_values_and_at_low_temperatures(rows, V):
    """p depends on the values' differences alone: rows of the type's lowest value are rows of equal ones at any temperature, and what the largest
    is does not cost digits (its difference from the others is exact here, and rounds once as it is divided)."""
    x, values, indices, _, up = made(rows, V, 5, F32)
    for tau in (0.5, 0.25, 2.0 ** -10):
        teachers = [torch.full_like(values, torch.finfo(F32).min), torch.full_like(values, torch.finfo(F32).max),
                    4096.0 + torch.arange(5, device="cuda").mul(-2.0 ** -11).expand_as(values)]
        alike = [torch.zeros_like(values), torch.zeros_like(values), teachers[2] - 4096.0]
        for teacher, same in zip(teachers, alike):
            leaf = x.detach().requires_grad_()
            losses = ldn.distillation_loss(leaf, teacher, indices, temperature=tau, reduction="none")
            want, bound, dx, off = oracle.loss_and_gradient(x, same, indices, None, tau, 0.0, up)
            assert head_oracle.near(losses.detach(), want, bound)
            # (a power below 2^-126, the smallest normal number, is 0: q is off by that much, and the gradient by up tau times it)
            assert head_oracle.near(torch.autograd.grad(losses, leaf, up)[0], dx, off + 2.0 ** -126 * tau * up.double().abs()[:, None])
