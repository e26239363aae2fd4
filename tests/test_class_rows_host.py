"""What label_log_probs and topk_distill refuse, in Python and at the C entry points, without a GPU."""
import ctypes

import pytest
import torch

import unet_amd
from unet_amd import TopKDistillLoss, label_log_probs, topk_distill, topk_distill_with_logits
from unet_amd import _lib
from unet_amd.class_rows import Rows


def refused(text, fn, *args, error=ValueError, **kw):
    with pytest.raises(error, match=text):
        fn(*args, **kw)


X = torch.zeros(4, 6)
LAB = torch.zeros(4, dtype=torch.int64)
V, IDX = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)


def test_label_log_probs_refuses():
    refused("fp32, bf16 or fp16", label_log_probs, X.double(), LAB)
    refused("fp32, bf16 or fp16", label_log_probs, [1.0], LAB)
    refused("class dimension", label_log_probs, X, LAB, dim=2)
    refused("class dimension", label_log_probs, torch.zeros(4), LAB)
    refused("0 classes", label_log_probs, torch.zeros(4, 0), LAB)
    refused("1048577 classes", label_log_probs, torch.zeros(1).expand(2, 1048577), LAB[:2])
    refused("top=7 of 6", label_log_probs, X, LAB, top=7)
    refused("top=-1", label_log_probs, X, LAB, top=-1)
    refused("top=65", label_log_probs, torch.zeros(2, 100), None, top=65)
    refused("temperature", label_log_probs, X, LAB, temperature=0.0)
    refused("temperature", label_log_probs, X, LAB, temperature=float("nan"))
    refused("temperature", label_log_probs, X, LAB, temperature=float("inf"))
    refused("expected shape", label_log_probs, X, LAB[:3])
    refused("expected shape", label_log_probs, X, LAB[:, None])
    refused("expected shape", label_log_probs, X, 3)
    refused("dtype", label_log_probs, X, LAB.float())
    refused("dtype", label_log_probs, X, LAB.to(torch.uint8))
    refused("HIP kernels only", label_log_probs, X, LAB, error=RuntimeError)


@pytest.mark.parametrize("fn", [topk_distill, topk_distill_with_logits])
def test_topk_distill_refuses(fn):
    refused("fp32, bf16 or fp16", fn, X.long(), V, IDX)
    refused("class dimension", fn, X, V, IDX, dim=5)
    refused("do not belong", fn, X, V[:3], IDX[:3])
    refused("do not belong", fn, X, V[0], IDX[0])
    refused("do not belong", fn, X, torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.int32))
    refused("do not belong", fn, torch.zeros(2, 400), torch.zeros(2, 257), torch.zeros(2, 257, dtype=torch.int32))
    refused("differ", fn, X, V, IDX[:, :2])
    refused("must be a tensor", fn, X, None, IDX)
    refused("dtype", fn, X, V.double(), IDX)
    refused("dtype", fn, X, V, IDX.float())
    refused("dtype", fn, X, V, IDX, weight=torch.zeros(4, dtype=torch.float64))
    refused("expected shape", fn, X, V, IDX, weight=torch.zeros(3))
    refused("reduction", fn, X, V, IDX, reduction="none")
    refused("temperature", fn, X, V, IDX, temperature=-1.0)
    refused("HIP kernels only", fn, X, V, IDX, error=RuntimeError)


def test_gradients_that_are_not_built_are_refused():
    x = X.clone().requires_grad_(True)
    refused("teacher's logits", topk_distill, x, V.clone().requires_grad_(True), IDX, error=NotImplementedError)
    refused("weights", topk_distill, x, V, IDX, weight=torch.ones(4, requires_grad=True), error=NotImplementedError)
    refused("temperature", TopKDistillLoss, 0.0)


def test_views_of_strided_logits():
    """row r = o*inner + i and class c of the view address the element that torch indexes"""
    base = torch.arange(2 * 3 * 4 * 5 * 2, dtype=torch.float32).reshape(2, 3, 4, 10)
    cases = [(base, 1), (base, -1), (base, 0), (base.permute(0, 3, 1, 2), 1), (base[:, :, 1:3], 1), (base[..., ::2], 3),
             (base[0, 0], 0), (base[0, 0, 0], 0), (base[:, :1], 1), (base.expand(2, 3, 4, 10), 2), (base[:1].expand(5, 3, 4, 10), 1)]
    for t, dim in cases:
        r = Rows(t, dim, "x")
        v = r.view
        flat = t.movedim(dim, -1).reshape(-1, t.shape[dim])
        assert v.outer * v.inner == len(flat) and v.classes == flat.shape[1]
        store = torch.as_strided(r.x, (r.x.untyped_storage().nbytes() // 4,), (1,), 0)
        at = r.x.storage_offset()
        for row in range(0, len(flat), 3):
            o, i = divmod(row, v.inner)
            for c in range(flat.shape[1]):
                assert store[at + o * v.so + i * v.si + c * v.sc] == flat[row, c]


def test_c_entry_points_refuse():
    lib = _lib.lib
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.cast(buf, ctypes.c_void_p)
    view = _lib.ClassView(4, 1, 6, 0, 1, 6, 0)
    ok = ctypes.byref(view)
    slots = _lib.Slots(p, p, 3, 0, 4)

    def no(text, name, *args):
        assert getattr(lib, name)(*args) == -1, name
        assert text in lib.uh_last_error().decode(), lib.uh_last_error()

    def probs(v=ok, x=p, lab=p, nb=8, top=0, t=1.0, lp=p, ent=p, tl=None, ti=None):
        return ("uh_label_log_probs", v, x, lab, nb, -100, top, t, lp, ent, tl, ti, None, None, 0, None)
    no("no view", *probs(v=None))
    no("null", *probs(x=None))
    no("null", *probs(ent=None))
    no("labels of 2 bytes", *probs(nb=2))
    no("top=65", *probs(top=65))
    no("top=7", *probs(top=7, tl=p, ti=p))
    no("null", *probs(top=3))
    no("temperature", *probs(t=0.0))
    no("temperature", *probs(t=5e-7))
    no("temperature", *probs(t=2e6))
    for bad in ((0, 1, 6, 0, 1, 6, 0), (4, 1, 6, 0, 1, 0, 0), (4, 1, 6, 0, 1, (1 << 20) + 1, 0), (4, 1, 6, 0, 1, 6, 3), (4, 1, 6, 0, -1, 6, 0),
                (1 << 20, 1 << 20, 6, 0, 1, 6, 0)):
        no("", *probs(v=ctypes.byref(_lib.ClassView(*bad))))
    other = ctypes.byref(_lib.ClassView(4, 1, 6, 0, 1, 7, 0))
    no("differs", "uh_label_log_probs_bwd", ok, other, p, p, 8, -100, 1.0, p, p, p, p, p, None)
    no("without labels", "uh_label_log_probs_bwd", ok, ok, p, None, 0, -100, 1.0, p, p, p, p, p, None)
    need = lib.uh_topk_distill_workspace(ok)
    assert need > 0 and lib.uh_topk_distill_workspace(other) > 0
    no("workspace", "uh_topk_distill", ok, p, ctypes.byref(slots), None, 1.0, 1.0, p, None, p, need - 1, None)
    no("no slots", "uh_topk_distill", ok, p, None, None, 1.0, 1.0, p, None, p, need, None)
    for bad in ((p, p, 0, 0, 4), (p, p, 257, 0, 4), (p, p, 3, 3, 4), (p, p, 3, 0, 2), (None, p, 3, 0, 4), (p, None, 3, 0, 4)):
        no("", "uh_topk_distill", ok, p, ctypes.byref(_lib.Slots(*bad)), None, 1.0, 1.0, p, None, p, need, None)
    no("temperature", "uh_topk_distill", ok, p, ctypes.byref(slots), None, float("nan"), 1.0, p, None, p, need, None)
    no("differs", "uh_topk_distill_bwd", ok, other, p, ctypes.byref(slots), None, 1.0, 1.0, p, p, p, None)
    no("null", "uh_topk_distill_bwd", ok, ok, p, ctypes.byref(slots), None, 1.0, 1.0, None, p, p, None)
    no("workspace", "uh_topk_distill_step", ok, ok, p, ctypes.byref(slots), None, 1.0, 1.0, 1.0, p, p, None, 0, None)


def test_public_names():
    for name in ("label_log_probs", "LabelLogProbs", "topk_distill", "topk_distill_with_logits", "teacher_targets", "TopKDistillLoss"):
        assert hasattr(unet_amd, name) and name in unet_amd.__all__
