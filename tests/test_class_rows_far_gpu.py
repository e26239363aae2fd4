"""Rows whose largest logit is far from zero (masks of -1e9, -1e10, -1e30 over whole rows, over their start or over a part of
them, ties at 3e9 or 1e25, the smallest temperatures): label_log_probs and topk_distill on every path against the plain 64-bit
implementation, with the tolerances of tests/class_rows_ref.py.  Those hold as they are: c (x - m) rounds the difference, c, the
product and T once each, and sums relative to the maximum itself need no correction."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from conftest import gpu_present            # noqa: E402

if not gpu_present():
    pytest.skip("needs a GPU", allow_module_level=True)

import class_rows_ref as ref                 # noqa: E402
import test_top_label_probs_gpu as probs     # noqa: E402
import test_topk_distill_gpu as dist         # noqa: E402
from unet_amd import label_log_probs, topk_distill, topk_distill_with_logits   # noqa: E402

DEV = probs.DEV
# type, temperature, and logits far at it on both sides of the border (|x| log2(e) / T = 2^24)
KINDS = [(torch.float32, 1.0, (-1e9, -1e10, -1e20, -1e30, 3e9, 1e12, 1e25, 2e7, -1.3e7, 1.1e7)),
         (torch.float32, 0.7, (-1e10, 1e12, -3e38, 1.7e7, -8.2e6, 8.1e6)),
         (torch.float32, 0.01, (-1e9, -1e5, 1.5e5, 116000.0)),
         (torch.bfloat16, 1.0, (-1e9, -1e10, -1e30, 3e9, 1e25, 2e7, -1.2e7)),
         (torch.bfloat16, 1e-6, (-1e10, 70.0, 11.5, -12.0, -0.3)),
         (torch.float16, 1e-6, (5000.0, -65504.0, -60000.0, 33.0, 11.6, -11.7)),
         (torch.float16, 1e-5, (5000.0, -65504.0, 120.0))]
IDS = [f"{str(d)[6:]}-{t}" for d, t, _ in KINDS]


def far_rows(c, dtype, fills, seed):
    """[rows, c]: per fill five rows; all of it, ties at it over classes a little and far below, its negative size as a mask over
    the first half, over the last quarter, and over all classes but one"""
    g = torch.Generator().manual_seed(seed)
    out = []
    for f in fills:
        a = abs(f)
        plain = torch.randn(5, c, generator=g, dtype=torch.float64) * 3
        ties = torch.full((c,), f, dtype=torch.float64)
        ties[1::3] -= a * 2.0 ** -7
        ties[2::5] -= a * 2.0 ** -22
        ties[3::7] -= a / 2
        start, end, one = plain[0].clone(), plain[1].clone(), torch.full((c,), -a, dtype=torch.float64)
        start[:(c + 1) // 2] = -a
        end[c - c // 4:] = -a
        one[c // 3] = plain[2, 0]
        out += [torch.full((c,), f, dtype=torch.float64), ties, start, end, one]
    big = torch.finfo(dtype).max
    return torch.stack(out).clamp(-big, big).to(dtype)


# rows [n, c], or maps of n images' worth of pixels; repeat: how often the rows occur (4097 and more: a thread walks its row)
PATHS = [("rows", 12, 1), ("rows", 53, 1), ("rows", 300, 1), ("rows", 3000, 1), ("rows", 9000, 1), ("rows", 40000, 1),
         ("rows", 131072, 1), ("rows", 5000, 60), ("maps", 12, 1), ("maps", 40, 3), ("maps", 90, 1), ("maps", 90, 300)]


def laid_out(layout, c, repeat, dtype, fills):
    x = far_rows(c, dtype, fills, c).repeat(repeat, 1)
    return x.to(DEV) if layout == "rows" else x.t().contiguous().view(1, c, -1, 5).to(DEV)


def check_gradient(x, labels, temperature):
    """The gradient of g log_prob + h entropy, g and h at once and h alone.  d = e (b z + a) = p [-g - h (ln p + H)] / T (+ g / T):
    the exponential e is flushed to 0 below 2^-126, the smallest normal number, and its factor, relative to p, is
    (|g| + |h| (|ln p| + H)) / T.  grad_tol counts the flushing for the first term alone, so that of the second is added
    (twice, for e relative to s >= 1 and the product's own flushing, as there)."""
    rows = ref.rows_of(x, 1)
    n, c = rows.shape
    lab = labels.reshape(-1).cpu()
    want = ref.label_probs(rows, lab, 0, temperature)
    lt, et = ref.log_tol(rows, c, temperature), ref.entropy_tol(rows, temperature)
    gen = torch.Generator().manual_seed(5)
    g, h = torch.randn(n, generator=gen), torch.randn(n, generator=gen) * 0.3
    for up in (g, None):
        leaf = x.detach().requires_grad_(True)
        got = label_log_probs(leaf, labels, temperature=temperature)
        outs, ups = [got.entropy], [h.to(DEV).view(labels.shape)]
        if up is not None:
            outs, ups = outs + [got.log_prob], ups + [up.to(DEV).view(labels.shape)]
        (dx,) = torch.autograd.grad(outs, leaf, ups)
        g64 = torch.zeros(n, dtype=torch.float64) if up is None else up.double()
        d = ref.label_probs_grad(rows, lab, temperature, None if up is None else g64, h.double())
        p = want["p"]
        lnp = torch.nan_to_num(want["logp"], neginf=0.0).abs()
        ha = (h.double().abs() / temperature)[:, None]
        hl = ha * (lnp + want["entropy"][:, None])
        tol = ref.grad_tol(x.dtype, d, p, g64.abs() / temperature, rows, c, temperature)
        tol = tol + torch.nan_to_num(p * hl * (lt + 2.0 ** -24 * 12)) + p * ha * torch.nan_to_num(lt + et[:, None]) + 2.0 ** -125 * hl
        ref.close(dx.movedim(1, -1).reshape(n, c), d, tol, "gradient")


@pytest.mark.parametrize("layout,c,repeat", PATHS)
@pytest.mark.parametrize("dtype,temperature,fills", KINDS, ids=IDS)
def test_label_log_probs(layout, c, repeat, dtype, temperature, fills):
    x = laid_out(layout, c, repeat, dtype, fills)
    labels = probs.labels_for(x, 1, 7)
    labels.view(-1)[::2] = c // 3                                # the class that is left, where one is
    probs.check(x, labels, top=min(c, 5), temperature=temperature, grads=False)
    probs.check(x, None, top=min(c, 12), temperature=temperature, grads=False)
    check_gradient(x, labels, temperature)


def slots_for(x, k):
    """a teacher with the student's masks that knows some of the classes: the student's best and others"""
    c = x.shape[1]
    best = torch.topk(x.float(), k - k // 2, dim=1).indices
    shape = list(x.shape)
    shape[1] = k // 2
    other = torch.randint(0, c, shape, generator=torch.Generator().manual_seed(c)).to(DEV)
    index = torch.cat([best, other], 1)
    value = x.gather(1, index)
    return value.contiguous(), index.int().contiguous()


@pytest.mark.parametrize("layout,c,repeat", PATHS)
@pytest.mark.parametrize("dtype,temperature,fills", KINDS, ids=IDS)
def test_topk_distill(layout, c, repeat, dtype, temperature, fills):
    """far students with near and far teachers; by weights, one row of the first ones at a time, so that no row's loss hides
    behind another's"""
    x = laid_out(layout, c, repeat, dtype, fills)
    value, index = slots_for(x, 6)
    near = probs.made(value.shape, torch.float32, c)
    rows = x.shape[0] if layout == "rows" else x.shape[2] * x.shape[3]
    for r in range(5 * len(fills)):
        weight = torch.zeros(rows, device=DEV)
        weight[r] = 1.0
        weight = weight if layout == "rows" else weight.view(1, *x.shape[2:])
        if c <= 300 or r % 3 == 0:
            for v in (value, near):
                loss = topk_distill(x, v, index, temperature, weight, "sum")
                one = [ref.rows_of(t, 1)[r:r + 1] for t in (x, v, index)]
                want, grad, _ = ref.distill(one[0], one[1], one[2].long(), temperature, None, 1.0)
                tol, _ = ref.distill_tols(one[0], one[1], one[2].long(), temperature, None, 1.0, grad, dtype)
                ref.close(loss, want, tol, f"loss of row {r}")
    dist.check(x, value, index, temperature, reduction="sum")
    dist.check(x, near, index, temperature, reduction="sum")


@pytest.mark.parametrize("dtype,temperature,fills", KINDS, ids=IDS)
def test_parts_that_nobody_waits_for(dtype, temperature, fills, monkeypatch):
    """the same bits whether a part's statistics arrive or are worked out by those who need them"""
    x = laid_out("rows", 70001, 1, dtype, fills)
    value, index = slots_for(x, 7)

    def run():
        leaf = x.detach().requires_grad_(True)
        loss = topk_distill(leaf, value, index, temperature)
        (dx,) = torch.autograd.grad(loss, leaf)
        return (topk_distill(x, value, index, temperature), loss.detach(), dx) + topk_distill_with_logits(x, value, index, temperature)

    want = run()
    monkeypatch.setenv("UNET_AMD_DISTILL_SPINS", "0")
    for a, b in zip(run(), want):
        assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("layout,c,repeat", PATHS)
@pytest.mark.parametrize("dtype,temperature,most", [(torch.float32, 0.7, -3e38), (torch.float32, 1e-3, -1e36), (torch.bfloat16, 1e-6, -1e33),
                                                    (torch.float32, 1.0, -3e38), (torch.bfloat16, 4.0, -3e38)])
def test_masked_labels_in_rows_past_the_largest_quotient(layout, c, repeat, dtype, temperature, most):
    """ln p of a class of -inf is -inf, also where the row's maximum over T is past the largest number"""
    x = torch.randn(20, c, generator=torch.Generator().manual_seed(9)).double()
    x[:10] = most
    x[:, 1::2] = -float("inf")
    x = x.to(dtype).repeat(repeat, 1)
    x = x.to(DEV) if layout == "rows" else x.t().contiguous().view(1, c, -1, 5).to(DEV)
    labels = probs.labels_for(x, 1, 7)
    labels.view(-1)[::3] = 1
    probs.check(x, labels, top=min(c, 5), temperature=temperature, grads=False)
    check_gradient(x, labels, temperature)
