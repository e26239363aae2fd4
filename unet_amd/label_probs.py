"""Log probabilities of given labels over class logits, with entropy and the top alternatives of every row.

    lp = label_log_probs(logits, labels, top=3)             # logits [B, C, H, W] or [rows, C], labels without the C
    loss = -lp.log_prob.mean() - 0.01 * lp.entropy.mean()   # cross entropy with an entropy term: differentiable
    value, index = lp.top_log_prob, lp.top_index            # a teacher's targets for `topk_distill`

The reference's losses know one-channel logits only (trainer/training_utils.py:105,146; the CrossEntropy term of
models/losses.py:58 is identically zero there); its networks take any number of output channels (models/unet.py:78,
models/lunext.py:185), and this is what such a head's logits are trained and judged with.
"""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import TOP_MAX, lib
from .class_rows import INT_BYTES, Rows, byref, checked_temperature, fp32_rows, refuse_tangents

LabelLogProbs = namedtuple("LabelLogProbs", "log_prob entropy top_log_prob top_index")


def _forward(r, labels, top, temperature, ignore_index, want_stats):
    dev, rows, f32 = r.device, r.row_shape, torch.float32
    entropy = torch.empty(rows, dtype=f32, device=dev)
    log_prob = top_lp = top_idx = stats = ws = None
    lab_ptr = lp_ptr = tl_ptr = ti_ptr = st_ptr = ws_ptr = None
    lab_bytes = 0
    if labels is not None:
        log_prob = torch.empty(rows, dtype=f32, device=dev)
        lab_ptr, lp_ptr, lab_bytes = labels.data_ptr(), log_prob.data_ptr(), INT_BYTES[labels.dtype]
    if top:
        shape = r.entries(top)
        top_lp = torch.empty(shape, dtype=f32, device=dev)
        top_idx = torch.empty(shape, dtype=torch.int32, device=dev)
        tl_ptr, ti_ptr = top_lp.data_ptr(), top_idx.data_ptr()
    if want_stats:
        stats = torch.empty((r.rows, 2), dtype=f32, device=dev)
        st_ptr = stats.data_ptr()
    if r.rows:
        v = byref(r.view)
        ws_bytes = lib.uh_label_log_probs_workspace(v, top)
        if ws_bytes:
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            ws_ptr = ws.data_ptr()
        r.call("uh_label_log_probs", v, r.x.data_ptr(), lab_ptr, lab_bytes, ignore_index, top, temperature, lp_ptr,
               entropy.data_ptr(), tl_ptr, ti_ptr, st_ptr, ws_ptr, ws_bytes)
    return log_prob, entropy, top_lp, top_idx, stats


class _LabelLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, r, labels, top, temperature, ignore_index):
        log_prob, entropy, top_lp, top_idx, stats = _forward(r, labels, top, temperature, ignore_index, True)
        ctx.save_for_backward(r.x, labels, stats, entropy)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_lp, top_idx)
        r.x = None                                # the saved tensors hold the logits, and let go of them
        ctx.args = (r, temperature, ignore_index)
        return log_prob, entropy, top_lp, top_idx

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, _g_top, _g_idx):
        if g_lp is None and g_ent is None:
            return (None,) * 6
        x, labels, stats, entropy = ctx.saved_tensors
        r, temperature, ignore_index = ctx.args
        dx, out_view = r.new_grad(x)
        if r.rows:
            g_lp, g_ent = fp32_rows(g_lp), fp32_rows(g_ent)
            r.bind("label_log_probs")
            lab = labels is not None
            r.call("uh_label_log_probs_bwd", byref(r.view), byref(out_view), x.data_ptr(),
                   labels.data_ptr() if lab else None, INT_BYTES[labels.dtype] if lab else 0, ignore_index, temperature,
                   stats.data_ptr(), entropy.data_ptr(), None if g_lp is None else g_lp.data_ptr(),
                   None if g_ent is None else g_ent.data_ptr(), dx.data_ptr())
        return dx, None, None, None, None, None


def label_log_probs(logits, labels=None, top=0, temperature=1.0, dim=1, ignore_index=-100):
    """(log_prob, entropy, top_log_prob, top_index) of every row of `logits`, with p = softmax(logits / temperature):

      log_prob      ln p[label], fp32, in the shape of `labels` (None without labels)
      entropy       -sum p ln p, fp32, the same shape
      top_log_prob  ln p of the `top` largest logits in falling order, with `top` in the place of the classes (None if
      top_index     top = 0), and their classes, int32.  Equal logits: the lowest class first.  Classes masked with -inf
                    are no alternatives; places left over hold -inf and -1

    logits: fp32, bf16 or fp16, classes in dimension `dim` (1, as the networks' heads give them; -1 for class-last
    tensors), up to 1048576 of them; any strides (dimensions in front of or behind the classes that no single stride
    walks are copied first).  labels: int64 or int32.  top: 0 to 64, at most the number of classes.

    A row whose label is `ignore_index` gives 0, 0 and no alternatives.  A label outside [0, C) makes its log_prob NaN
    (there is no check that would have to wait for the device).  A row that holds a NaN or +inf gives NaN and indices -1;
    a row of nothing but -inf gives log_prob -inf, entropy 0 and no alternatives.

    log_prob and entropy are differentiable with respect to the logits (once, in reverse mode: logits with a forward-mode
    tangent are refused); the alternatives are not.  The gradient has the logits' type; rows that are ignored or nothing but -inf get zeros."""
    what = "label_log_probs"
    r = Rows(logits, dim, what)
    refuse_tangents(what, logits)
    temperature = checked_temperature(temperature, what)
    top = int(top)
    if not 0 <= top <= min(TOP_MAX, r.classes):
        raise ValueError(f"{what}: top={top} of {r.classes} classes (0 to {min(TOP_MAX, r.classes)})")
    if labels is not None:
        labels = r.per_row(labels, f"{what}: labels", INT_BYTES)
    r.bind(what)
    if torch.is_grad_enabled() and logits.requires_grad:
        return LabelLogProbs(*_LabelLogProbsFn.apply(logits, r, labels, top, temperature, int(ignore_index)))
    return LabelLogProbs(*_forward(r, labels, top, temperature, int(ignore_index), False)[:4])
