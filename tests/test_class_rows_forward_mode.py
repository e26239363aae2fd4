"""A forward-mode tangent is refused and not left behind: the kernels have no rule for it."""
import pytest
import torch
from torch.autograd import forward_ad

from unet_amd import label_log_probs, teacher_targets, topk_distill

X = torch.zeros(4, 6)
LAB = torch.zeros(4, dtype=torch.int64)
V, IDX, W = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32), torch.ones(4)


def test_tangents_are_refused():
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: label_log_probs(dual(X), LAB), lambda: teacher_targets(dual(X), 2), lambda: topk_distill(dual(X), V, IDX),
                     lambda: topk_distill(X, dual(V), IDX), lambda: topk_distill(X, V, IDX, weight=dual(W))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):       # which tangents outlive
                call()


def test_jvp_is_refused():
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: label_log_probs(x, LAB).log_prob, (X,), (torch.ones_like(X),))


def test_tensors_without_a_tangent_pass_the_check():
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="HIP kernels only"):
        label_log_probs(X, LAB)
