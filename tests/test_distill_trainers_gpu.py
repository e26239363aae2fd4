"""Criteria over a teacher's targets in the trainers: a subclass of TopKDistillLoss with a term of its own, targets with weights,
and a GradScaler, each against the same model's autograd."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from conftest import gpu_present            # noqa: E402

if not gpu_present():
    pytest.skip("needs a GPU", allow_module_level=True)

import unet_amd                              # noqa: E402
from unet_amd import TopKDistillLoss, label_log_probs   # noqa: E402
from unet_amd.dp import DataParallelTrainer, LUNeXtTrainer   # noqa: E402

DEV = torch.device("cuda", 0)
CLASSES = 4


class WithHardLabels(TopKDistillLoss):
    """the teacher's best class as a label next to its distribution"""

    def forward(self, logits, targets):
        hard = label_log_probs(logits, targets[1].select(1, 0))
        return super().forward(logits, targets) - 3.0 * hard.log_prob.mean()


def made(weights):
    g = torch.Generator().manual_seed(3)
    images = torch.rand(2, 3, 32, 48, generator=g).to(DEV)
    scores = torch.randn(2, CLASSES, 32, 48, generator=g).to(DEV)
    value, index = torch.topk(scores, 2, dim=1)
    targets = (value.contiguous(), index.int().contiguous())
    return images, targets + ((torch.rand(2, 32, 48, generator=g).to(DEV),) if weights else ())


@pytest.mark.parametrize("criterion", [TopKDistillLoss, WithHardLabels])
@pytest.mark.parametrize("weights", [False, True])
def test_light_network(criterion, weights):
    images, targets = made(weights)
    torch.manual_seed(0)
    student = unet_amd.LUNeXt(3, CLASSES).to(DEV).train()
    twin, crit = copy.deepcopy(student), criterion(2.0)
    want = crit(twin(images), targets)
    want.backward()
    trainer = LUNeXtTrainer(student, criterion=crit, standalone=True)
    got = trainer.train_step(images, targets)
    assert torch.allclose(got, want.detach(), rtol=1e-5)
    a, b = trainer.grads.views["final_conv.weight"], twin.final_conv.weight.grad
    assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * b.abs().max().item())


@pytest.mark.parametrize("criterion", [TopKDistillLoss, WithHardLabels])
@pytest.mark.parametrize("scaled", [False, True])
def test_heavy_network(criterion, scaled):
    """with a GradScaler the gradients in the buckets are those of the scaled loss; the backward passes are the same kernels behind
    gradients of the logits that differ by a few roundings of fp32, which bf16 activations turn into steps of 2^-8 here and there"""
    images, targets = made(True)
    torch.manual_seed(0)
    student = unet_amd.UNet(3, CLASSES).to(DEV).train()
    twin, crit = copy.deepcopy(student), criterion(2.0)
    want = crit(twin(images), targets)
    want.backward()
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0) if scaled else None
    trainer = DataParallelTrainer(student, criterion=crit, standalone=True)
    got = trainer.train_step(images, targets, scaler=scaler)
    assert torch.allclose(got, want.detach(), rtol=1e-5)
    for name in ("final_conv.weight", "conv_up4_2.weight"):
        a, b = trainer.buckets.views[name].float() / (1024.0 if scaled else 1.0), dict(twin.named_parameters())[name].grad
        cos = (a.flatten() @ b.flatten()) / (a.norm() * b.norm())
        assert cos > 0.999 and abs((a.norm() / b.norm()).item() - 1.0) < 1e-2, name
    assert torch.isfinite(trainer.train_step(images, targets, scaler=scaler))


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_a_ranks_share_of_the_gradient(reduction):
    """one of two ranks seeds its backward pass with half of its own loss's gradient (a power of two: the same bits, halved)"""
    _, targets = made(True)
    trainer = LUNeXtTrainer(unet_amd.LUNeXt(3, CLASSES).to(DEV).train(), criterion=TopKDistillLoss(2.0, reduction), standalone=True)
    logits = torch.randn(2, CLASSES, 32, 48, generator=torch.Generator().manual_seed(4)).to(DEV)
    loss, whole = trainer._loss(logits, targets)
    trainer.world = 2
    again, half = trainer._loss(logits, targets)
    assert torch.equal(loss, again) and torch.equal(whole, half * 2.0)
