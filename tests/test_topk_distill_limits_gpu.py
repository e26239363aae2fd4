"""topk_distill where a class that the teacher names is masked with the type's lowest value: the loss without T^2 is past the
largest fp32 number for T < 1, the loss itself is not."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from conftest import gpu_present            # noqa: E402

if not gpu_present():
    pytest.skip("needs a GPU", allow_module_level=True)

import class_rows_ref as ref                 # noqa: E402
import test_topk_distill_gpu as dist         # noqa: E402
from unet_amd import topk_distill, topk_distill_with_logits   # noqa: E402

DEV = dist.DEV


def flushed(x, v, index, temperature, *_):
    """What a loss may lose where a slot's exponential, relative to the largest one's, is below 2^-126, the smallest normal fp32
    number, and counts as 0: a t_k of at most that times |ln t_k - ln p| T^2, which is of account beside a logit of -3e38."""
    logt, logp = ref.softmax_parts(v, temperature)[0], ref.softmax_parts(x, temperature)[0].gather(1, index)
    return (2.0 ** -126 * torch.where(logt < -126 * math.log(2.0), (logt - logp).abs(), 0.0)).sum() * temperature ** 2


# a thread's rows side by side, 16 lanes, a wave, a workgroup, parts; classes that lie apart: a thread's, 256 lanes', walked
@pytest.mark.parametrize("shape", [(3, 12), (3, 40), (3, 300), (3, 3000), (600, 9000), (3, 40000), (3, 12, 2, 2), (3, 90, 2, 2),
                                   (3, 90, 64, 32)])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 0.25, 0.01, 3.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_classes_masked_with_the_lowest_value(shape, temperature, dtype):
    """the loss of one row at a time: its neighbours' would pass the largest number with it"""
    big = torch.finfo(dtype).max
    x = dist.made(shape, dtype, 81)
    value, index = dist.targets_for(x, 3, 81)
    masked = index[:, 1:2].long()
    x.scatter_(1, masked, -big)
    high = x.clone()
    high.scatter_(1, index[:, :1].long(), big)                    # the difference of two logits overflows as well
    for y in (x, high):
        rows, vr, ir = ref.rows_of(y, 1), ref.rows_of(value, 1), ref.rows_of(index, 1).long()
        for r in (0, 2):
            weight = torch.zeros(len(rows), device=DEV)
            weight[r] = 1.0
            weight = weight.view(index[:, 0].shape)
            one = (rows[r:r + 1], vr[r:r + 1], ir[r:r + 1], temperature, None, 1.0)
            want, grad, _ = ref.distill(*one)
            tol = ref.distill_tols(*one, grad, dtype)[0] + flushed(*one)
            ref.close(topk_distill(y, value, index, temperature, weight, "sum"), want, tol, "loss")
            loss, _ = topk_distill_with_logits(y, value, index, temperature, weight, "sum")
            ref.close(loss, want, tol, "loss of the step")
