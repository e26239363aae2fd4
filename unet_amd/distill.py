"""Distillation from a teacher's top logits: the light network (LUNeXt) learns the heavy one's class probabilities from a
few stored logits per pixel instead of its whole output.

    targets = teacher_targets(teacher(images), top=4)                 # (values, classes): [B, 4, H, W]
    loss = topk_distill(student(images), *targets, temperature=2.0)   # differentiable
    trainer = LUNeXtTrainer(student, criterion=TopKDistillLoss(temperature=2.0))
    trainer.train_step(images, targets)                               # value and gradient from one kernel pass

The reference trains every network from the masks alone (trainer/training_utils.py:139-160).
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import SLOTS_MAX, lib
from .class_rows import DTYPE_CODE, INT_BYTES, Rows, byref, checked_temperature, fp32_rows, refuse_tangents
from .label_probs import label_log_probs


class _Targets:
    """the checked slots and weights of a call, dense in the rows' order"""
    __slots__ = ("value", "index", "weight", "slots")

    def __init__(self, r, top_logits, top_index, weight, what):
        for t, name in ((top_logits, "top_logits"), (top_index, "top_index")):
            if not torch.is_tensor(t):
                raise ValueError(f"{what}: {name} must be a tensor")
        k = top_logits.shape[r.dim] if top_logits.dim() == len(r.row_shape) + 1 else 0
        if not 0 < k <= SLOTS_MAX or top_logits.shape != r.entries(k):
            raise ValueError(f"{what}: top_logits {tuple(top_logits.shape)} do not belong to logits {tuple(r.x.shape)} with "
                             f"the classes in dimension {r.dim} (1 to {SLOTS_MAX} slots)")
        if top_index.shape != top_logits.shape:
            raise ValueError(f"{what}: top_index {tuple(top_index.shape)} and top_logits {tuple(top_logits.shape)} differ")
        if torch.is_grad_enabled() and top_logits.requires_grad:
            raise NotImplementedError(f"{what}: the gradient with respect to the teacher's logits is not built")
        if weight is not None and torch.is_grad_enabled() and torch.is_tensor(weight) and weight.requires_grad:
            raise NotImplementedError(f"{what}: the gradient with respect to the weights is not built")
        self.value = r.same_device(top_logits, f"{what}: top_logits", DTYPE_CODE)
        self.index = r.same_device(top_index, f"{what}: top_index", INT_BYTES)
        self.weight = None if weight is None else r.per_row(weight, f"{what}: weight", (torch.float32,))
        self.slots = _slots(self.value, self.index, k)

    @property
    def weight_ptr(self):
        return None if self.weight is None else self.weight.data_ptr()


def _slots(value, index, k):
    return _lib.Slots(value.data_ptr(), index.data_ptr(), k, DTYPE_CODE[value.dtype], INT_BYTES[index.dtype])


def _forward(r, t, temperature, scale, want_stats):
    loss = torch.empty((), dtype=torch.float32, device=r.device)
    stats = torch.empty((r.rows, 2), dtype=torch.float32, device=r.device) if want_stats else None
    ws_bytes = lib.uh_topk_distill_workspace(byref(r.view))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=r.device)
    r.call("uh_topk_distill", byref(r.view), r.x.data_ptr(), byref(t.slots), t.weight_ptr, temperature, scale,
           loss.data_ptr(), stats.data_ptr() if want_stats else None, ws.data_ptr(), ws_bytes)
    return loss, stats


class _TopKDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, r, t, temperature, scale):
        loss, stats = _forward(r, t, temperature, scale, True)
        ctx.save_for_backward(r.x, t.value, t.index, t.weight, stats)
        r.x = None                                # the saved tensors hold the logits, and let go of them
        ctx.args = (r, temperature, scale)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        x, value, index, weight, stats = ctx.saved_tensors
        r, temperature, scale = ctx.args
        dx, out_view = r.new_grad(x)
        g = fp32_rows(gout)
        r.bind("topk_distill")
        r.call("uh_topk_distill_bwd", byref(r.view), byref(out_view), x.data_ptr(),
               byref(_slots(value, index, value.shape[r.dim])), None if weight is None else weight.data_ptr(),
               temperature, scale, g.data_ptr(), stats.data_ptr(), dx.data_ptr())
        return dx, None, None, None, None


def _scale(r, reduction, what):
    if reduction not in ("mean", "sum"):
        raise ValueError(f"{what}: reduction {reduction!r} (mean or sum)")
    return 1.0 / max(r.rows, 1) if reduction == "mean" else 1.0


def topk_distill(logits, top_logits, top_index, temperature=1.0, weight=None, reduction="mean", dim=1):
    """The distillation loss of a student's `logits` against a teacher's slots, a 0-dim fp32 tensor, differentiable with
    respect to the logits (once, in reverse mode: forward-mode tangents are refused):

        t = softmax over the slots of top_logits / T,   p = softmax over the classes of logits / T
        loss = mean (or sum) over the rows of  weight * T^2 * sum_k t_k (ln t_k - ln p[top_index_k])

    logits: fp32, bf16 or fp16, classes in dimension `dim`, any strides; top_logits, top_index: 1 to 256 slots in the place
    of the classes, values in any of the three types (logits or log probabilities), classes as int32 or int64.  A negative
    index is a free slot (`teacher_targets` leaves those where there are fewer classes to name).  A class named twice
    counts twice.  weight: fp32 per row or None.

    Rows of weight 0 and rows without a filled slot count as 0 whatever they hold, and get zero gradients; the mean divides
    by the number of all rows.  A slot whose t_k is below 2^-126, the smallest normal fp32 number, counts as t_k = 0, also where
    the student gives its class no probability.  A class index past the last one, or a NaN, makes the loss NaN.  Without any row the loss is
    0.  The loss is summed in a fixed order: equal inputs give equal bits."""
    what = "topk_distill"
    r = Rows(logits, dim, what)
    temperature = checked_temperature(temperature, what)
    t = _Targets(r, top_logits, top_index, weight, what)
    refuse_tangents(what, logits, top_logits, weight)
    scale = _scale(r, reduction, what)
    r.bind(what)
    if r.rows == 0:
        return logits.float().sum()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TopKDistillFn.apply(logits, r, t, temperature, scale)
    return _forward(r, t, temperature, scale, False)[0]


def topk_distill_with_logits(logits, top_logits, top_index, temperature=1.0, weight=None, reduction="mean", grad_scale=1.0,
                             dim=1):
    """(topk_distill(...), grad_scale * its gradient with respect to the logits) without autograd, from one pass over the
    logits: what a training step that runs its own backward pass takes (as bce_with_logits and cldice_with_logits)."""
    what = "topk_distill_with_logits"
    r = Rows(logits, dim, what)
    temperature = checked_temperature(temperature, what)
    with torch.no_grad():
        t = _Targets(r, top_logits, top_index, weight, what)
        scale = _scale(r, reduction, what)
        r.bind(what)
        if r.rows == 0:
            return torch.zeros((), dtype=torch.float32, device=r.device), torch.empty_like(r.x)
        dx, out_view = r.new_grad(r.x)
        loss = torch.empty((), dtype=torch.float32, device=r.device)
        ws_bytes = lib.uh_topk_distill_workspace(byref(r.view))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=r.device)
        r.call("uh_topk_distill_step", byref(r.view), byref(out_view), r.x.data_ptr(), byref(t.slots), t.weight_ptr,
               temperature, scale, float(grad_scale), loss.data_ptr(), dx.data_ptr(), ws.data_ptr(), ws_bytes)
    return loss, dx


def teacher_targets(logits, top, dim=1):
    """(values, classes) of the `top` largest of a teacher's logits in every row, as topk_distill takes them: fp32 log
    probabilities (they differ from the logits by a constant per row, which the loss does not see) and int32 classes."""
    with torch.no_grad():
        lp = label_log_probs(logits, top=top, dim=dim)
    return lp.top_log_prob, lp.top_index


class TopKDistillLoss(nn.Module):
    """topk_distill as a criterion: forward(logits, targets) with targets = (top_logits, top_index) or (top_logits,
    top_index, weight).  The trainers (DataParallelTrainer, LUNeXtTrainer) take value and gradient from one pass
    (`value_and_grad`); anything else may call it like any differentiable loss, and so do the trainers with a subclass, whose
    forward may add terms of its own."""

    def __init__(self, temperature=1.0, reduction="mean", dim=1):
        super().__init__()
        self.temperature, self.reduction, self.dim = checked_temperature(temperature, "TopKDistillLoss"), reduction, dim

    def forward(self, logits, targets):
        return topk_distill(logits, targets[0], targets[1], self.temperature, *targets[2:3], reduction=self.reduction,
                            dim=self.dim)

    def value_and_grad(self, logits, targets, grad_scale=1.0):
        return topk_distill_with_logits(logits, targets[0], targets[1], self.temperature, *targets[2:3],
                                        reduction=self.reduction, grad_scale=grad_scale, dim=self.dim)
