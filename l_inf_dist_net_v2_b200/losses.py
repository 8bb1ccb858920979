"""Training losses of the reference driver (main.py:304-330), as callables `loss(outputs, worst_outputs, targets)`
on what the models return: `hinge` and `mixture` act on the margins of `MLPModel`, `crossentropy` on the
worst-case logit differences of `HybridModel`.  `distillation` (not in the reference) is for any model's logits and a teacher's."""
import math

import torch.nn.functional as F

from . import norm_dist_cuda as _C

__all__ = ["hinge", "crossentropy", "mixture", "distillation", "distillation_loss"]

_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


class hinge:
    """(1 - mix) * mean over samples of the largest positive margin + mix * mean of all positive margins."""

    def __init__(self, mix=0.25):
        self.mix = mix

    def __call__(self, outputs, worst_outputs, targets):
        ext = _C.native() if worst_outputs.is_cuda and isinstance(self.mix, (int, float)) else None
        loss = None if ext is None else ext.hinge(worst_outputs, self.mix)  # one kernel; None: not for it
        if loss is not None:
            return loss
        pos = worst_outputs.clamp(min=0)
        return (1 - self.mix) * pos.max(dim=1)[0].mean() + self.mix * pos.mean()


class crossentropy:
    def __init__(self, mix=0):
        self.mix = mix

    def __call__(self, outputs, worst_outputs, targets):
        robust = F.cross_entropy(worst_outputs, targets)
        if self.mix == 0:
            return robust
        return (1 - self.mix) * robust + self.mix * F.cross_entropy(outputs, targets)


class mixture:
    """Clipped hinge on the margins plus lam * cross-entropy on the logits; lam decays geometrically from lam0 to
    lam_end as `update(ratio)` is called with ratio going from 0 to 1."""

    def __init__(self, lam0=0.1, lam_end=0.001, clip=1):
        self.lam_start = lam0
        self.lam_end = lam_end
        self.lam = lam0
        self.speed = math.log(lam_end / lam0)
        self.clip = clip

    def update(self, ratio):
        self.lam = self.lam_start * math.exp(self.speed * ratio)

    def __call__(self, outputs, worst_outputs, targets):
        pos = worst_outputs.clamp(min=0, max=self.clip)
        return pos.max(dim=1)[0].mean() + self.lam * F.cross_entropy(outputs, targets)


def distillation_loss(logits, teacher_values, teacher_indices, targets=None, temperature=1.0, mix=0.0, reduction="mean"):
    """Distillation from a teacher's top logits: per row of `logits` (..., classes)

        (1 - mix) temperature^2 sum p (log p - log q) + mix cross_entropy(logits, target),

    p = softmax(teacher_values / temperature) over the row's entries and q = softmax(logits / temperature) over all classes, with the
    gradient of the logits (the teacher has none).  `teacher_values` and `teacher_indices` (..., k), k up to 1024, say which classes the
    entries are of, in any order; an entry with an index below 0 is absent.  Entries of one class add up beside log q
    and in the gradient, while log p is each entry's own: a class that is listed several times lowers the loss by a number that does
    not depend on the logits (twice alike, with nothing else to choose: -temperature^2 log 2).  A row without entries has no
    first term, a row with a target below 0 no second; a term that `mix` gives no weight is none, infinite ones too.  An index or target
    beyond the classes makes its row's loss and gradient not-a-numbers.

    reduction: "mean" over all rows, "sum" or "none"; the loss is float32.  Logits are float32, float16 or bfloat16 and may hold minus
    infinity for classes that are no choice; sums have 32 bits and are made in one pass over the logits each way."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, not {reduction!r}")
    if mix and targets is None:
        raise ValueError("a mix with the labels' cross-entropy needs targets")
    ext = _C.native()
    if ext is None:
        raise RuntimeError("distillation_loss needs the compiled binding (python l_inf_dist_net_v2_b200/build.py) and runs under no "
                           "function transform and not in torch.compile")
    return ext.distillation_loss(logits, teacher_values, teacher_indices, targets if mix else None, temperature, mix,
                                 _REDUCTIONS[reduction])


class distillation:
    """`distillation_loss` as a training loss: loss(outputs, teacher, targets) with `teacher` a (values, indices) pair, as
    `teacher_logits.topk(k)` gives it."""

    def __init__(self, temperature=4.0, mix=0.1):
        self.temperature = temperature
        self.mix = mix

    def __call__(self, outputs, teacher, targets=None):
        return distillation_loss(outputs, teacher[0], teacher[1], targets, self.temperature, self.mix)
