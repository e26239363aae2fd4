"""topk_distill, topk_distill_with_logits, teacher_targets and TopKDistillLoss against a plain 64-bit implementation
(tests/class_rows_ref.py), and a light network taught by a heavy one."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from conftest import gpu_present            # noqa: E402

if not gpu_present():
    pytest.skip("needs a GPU", allow_module_level=True)

import class_rows_ref as ref                 # noqa: E402
import unet_amd                              # noqa: E402
from unet_amd import TopKDistillLoss, label_log_probs, teacher_targets, topk_distill, topk_distill_with_logits   # noqa: E402

DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = math.inf, math.nan


def made(shape, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype).to(DEV)


def targets_for(x, k, seed, dim=1, dtype=torch.float32, index=torch.int32):
    teacher = x.float() + made(x.shape, torch.float32, seed + 50, 1.0)
    v, i = torch.topk(teacher, k, dim=dim)
    return v.to(dtype).contiguous(), i.to(index).contiguous()


def check(x, v, i, temperature=1.0, weight=None, reduction="mean", grad_scale=1.0, dim=1):
    rows = ref.rows_of(x, dim)
    n, c = rows.shape
    vr, ir = ref.rows_of(v, dim), ref.rows_of(i, dim).long()
    w = None if weight is None else weight.reshape(-1).cpu()
    scale = 1.0 / n if reduction == "mean" else 1.0
    loss, grad, _ = ref.distill(rows, vr, ir, temperature, w, scale)
    lt, gt = ref.distill_tols(rows, vr, ir, temperature, w, scale, grad, x.dtype)
    back = lambda d: d.detach().movedim(dim, -1).reshape(n, c)                           # noqa: E731
    got = topk_distill(x, v, i, temperature, weight, reduction, dim)
    assert got.dtype == torch.float32 and got.shape == ()
    ref.close(got, loss, lt, "loss")
    leaf = x.detach().requires_grad_(True)
    again = topk_distill(leaf, v, i, temperature, weight, reduction, dim)
    assert torch.equal(again.detach(), got) or bool(got.isnan())
    (dx,) = torch.autograd.grad(again, leaf)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    ref.close(back(dx), grad, gt, "gradient")
    value, step = topk_distill_with_logits(x, v, i, temperature, weight, reduction, grad_scale, dim)
    assert step.dtype == x.dtype and step.shape == x.shape
    ref.close(value, loss, lt, "loss of the step")
    loss2, grad2, _ = ref.distill(rows, vr, ir, temperature, w, scale)
    _, gt2 = ref.distill_tols(rows, vr, ir, temperature, w, scale * abs(grad_scale), grad * grad_scale, x.dtype)
    ref.close(back(step), grad * grad_scale, gt2, "gradient of the step")
    return got, dx


ROWS = [(1, 1, 1), (1, 2, 1), (5, 3, 2), (130, 7, 3), (257, 19, 4), (64, 64, 8), (33, 65, 5), (7, 100, 20), (19, 129, 64), (3, 511, 7),
        (6, 513, 33), (5, 1000, 50), (4, 2049, 3), (3, 4097, 100), (2, 5003, 4), (2, 8191, 65), (1, 16385, 9), (3, 32000, 64),
        (2, 33001, 128), (1, 70001, 5), (2, 131072, 100), (1, 140003, 256)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,c,k", ROWS)
def test_rows(n, c, k, dtype):
    x = made((n, c), dtype, n * 31 + c)
    check(x, *targets_for(x, k, c), temperature=2.0, reduction="sum")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,k", [((1, 2, 1, 3), 2), ((2, 1, 5, 7), 1), ((3, 8, 9, 11), 4), ((2, 19, 33, 21), 3), ((1, 21, 64, 64), 4),
                                     ((1, 64, 8, 9), 9), ((1, 65, 16, 17), 8), ((2, 100, 7, 5), 64), ((1, 300, 4, 33), 5),
                                     ((1, 2000, 3, 5), 20)])
def test_class_maps(shape, k, dtype):
    x = made(shape, dtype, sum(shape))
    check(x, *targets_for(x, k, 3, dtype=dtype, index=torch.int64), temperature=0.75, reduction="sum", grad_scale=2.5)


@pytest.mark.parametrize("shape", [(300, 12), (40, 200), (30, 3000), (6, 40000), (3, 9, 12, 11)])
def test_weights_and_mean(shape):
    x = made(shape, torch.float32, 4)
    v, i = targets_for(x, 5, 4)
    rows = v.movedim(1, -1).shape[:-1]
    w = torch.rand(rows, generator=torch.Generator().manual_seed(3)).to(DEV)
    w.view(-1)[::4] = 0.0
    check(x, v, i, 2.0, w)
    check(x, v, i, 2.0, w, "sum", grad_scale=-0.5)
    # rows of weight 0 may hold anything: NaN logits, NaN slots, classes that do not exist
    off = (w == 0).unsqueeze(1)
    xx, vv = x.masked_fill(off, NAN), v.masked_fill(off, NAN)
    ii = i.masked_fill(off, 10 ** 8)
    a, da = check(xx, vv, ii, 2.0, w)
    assert torch.isfinite(a) and torch.isfinite(da).all()


@pytest.mark.parametrize("shape", [(12, 9), (12, 64), (12, 200), (12, 1500), (12, 9000), (12, 40000), (3, 9, 2, 2), (3, 70, 2, 2)])
def test_free_slots_and_repeated_classes(shape):
    x = made(shape, torch.float32, 5)
    v, i = targets_for(x, 8, 5)
    vr, ir = v.movedim(1, -1).reshape(-1, 8).clone(), i.movedim(1, -1).reshape(-1, 8).clone()
    ir[0, 5:] = -1                    # some free slots, with values in them
    ir[1] = -1                        # no slot at all
    ir[2] = ir[2, 0]                  # one class in all of them
    ir[3, 4:] = ir[3, :4]
    vr[4, 3:] = -INF                  # a teacher without probability for them
    vr[5] = -INF
    vr[6, 0] = torch.finfo(torch.float32).max
    vr[7] = torch.finfo(torch.float32).min
    ir[8, ::2] = -5
    shape_back = v.movedim(1, -1).shape
    v, i = (t.reshape(shape_back).movedim(-1, 1).contiguous() for t in (vr, ir))
    for t in (1.0, 0.5, 4.0):
        got, dx = check(x, v, i, t, reduction="sum")
    assert torch.isfinite(got)


@pytest.mark.parametrize("shape", [(12, 9), (12, 200), (12, 9000), (12, 40000), (3, 9, 2, 2), (3, 70, 2, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_masked_and_undefined_students(shape, dtype):
    x = made(shape, dtype, 6)
    v, i = targets_for(x, 4, 6)
    r = x.movedim(1, -1).reshape(-1, shape[1]).clone()
    ir = i.movedim(1, -1).reshape(-1, 4)
    keep = torch.zeros_like(r, dtype=torch.bool).scatter_(1, ir.long(), True)
    r[0] = r[0].masked_fill(~keep[0], -INF)              # only the teacher's classes are left
    r[1] = r[1].masked_fill(~keep[1], torch.finfo(dtype).min)
    r[2] = torch.finfo(dtype).min                        # uniform
    x = r.reshape(x.movedim(1, -1).shape).movedim(-1, 1).contiguous()
    got, _ = check(x, v, i, 1.0, reduction="sum")
    assert torch.isfinite(got)
    for row, fill in ((3, NAN), (4, INF), (5, -INF)):    # undefined rows; a student without any class left
        rr = r.clone()
        if fill == -INF:
            rr[row] = fill
        else:
            rr[row, shape[1] // 2] = fill
        y = rr.reshape(x.movedim(1, -1).shape).movedim(-1, 1).contiguous()
        got, dx = check(y, v, i, 1.0, reduction="sum")
        assert not torch.isfinite(got)
    rr = r.clone()
    rr[6, ir[6, 0].long()] = -INF                        # a class the teacher believes in is masked: the loss is inf
    y = rr.reshape(x.movedim(1, -1).shape).movedim(-1, 1).contiguous()
    got, dx = check(y, v, i, 1.0, reduction="sum")
    assert got.item() == INF and torch.isfinite(dx.float()).all()


@pytest.mark.parametrize("shape", [(5, 9), (5, 200), (5, 9000), (3, 40000), (1, 9, 2, 2), (1, 70, 2, 2)])
def test_undefined_teachers(shape):
    x = made(shape, torch.float32, 7)
    v, i = targets_for(x, 3, 7)
    for what in ("nan", "inf", "index", "nan in a free slot"):
        vv, ii = v.clone(), i.clone()
        vr, ir = vv.movedim(1, -1), ii.movedim(1, -1)
        at = (1, 1) if len(shape) == 2 else (0, 0, 1, 1)
        if what == "index":
            ir[at] = shape[1]
        else:
            vr[at] = INF if what == "inf" else NAN
        if what == "nan in a free slot":
            ir[at] = -1
        got, dx = check(x, vv, ii, 1.0, reduction="sum")
        assert math.isnan(got.item())
        bad = dx.movedim(1, -1).reshape(-1, shape[1])
        assert torch.isnan(bad[1]).all() and torch.isfinite(bad[0]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides(dtype):
    last = made((2, 6, 10, 300), dtype, 8).permute(0, 3, 1, 2)
    check(last, *targets_for(last, 4, 1), reduction="sum")
    small = made((3, 5, 7, 11), dtype, 9).permute(0, 3, 1, 2)
    check(small, *targets_for(small, 4, 1), reduction="sum")
    for c in (21, 333, 5001):
        wide = made((9, c + 13), dtype, 10)
        for off in (0, 1, 5):
            rows = wide[:, off:off + c]
            check(rows, *targets_for(rows, 4, 1), reduction="sum")
    t = made((40, 9), dtype, 11).t()
    check(t, *targets_for(t, 4, 1), reduction="sum")
    e = made((1, 40), dtype, 12).expand(5, 40)
    check(e, *targets_for(e, 4, 1), reduction="sum")
    s = made((2, 8, 9, 10), dtype, 13)[:, 1:6, 2:7, ::3]
    check(s, *targets_for(s, 3, 1), reduction="sum")
    seq = made((2, 3, 130), dtype, 14)
    check(seq, *targets_for(seq, 3, 1, dim=-1), reduction="sum", dim=-1)
    v, i = targets_for(seq, 3, 1, dim=-1)
    check(seq, v.transpose(0, 1).contiguous().transpose(0, 1), i.repeat(1, 1, 2)[..., ::2][..., [0, 1, 2]], reduction="sum", dim=-1)


def test_offsets_past_32_bits():
    step = 1_100_000_000
    buf = torch.empty(2 * step + 2000, dtype=torch.bfloat16, device=DEV)
    rows = buf.as_strided((3, 1000), (step, 1))
    rows.copy_(made((3, 1000), torch.bfloat16, 4))
    check(rows, *targets_for(rows.contiguous(), 5, 1))


def test_no_rows():
    x = torch.empty(0, 5, device=DEV, requires_grad=True)
    v, i = torch.empty(0, 2, device=DEV), torch.empty(0, 2, dtype=torch.int32, device=DEV)
    loss = topk_distill(x, v, i)
    assert loss.item() == 0.0
    (dx,) = torch.autograd.grad(loss, x)
    assert dx.shape == x.shape
    loss, dx = topk_distill_with_logits(x.detach(), v, i)
    assert loss.item() == 0.0 and dx.shape == x.shape


@pytest.mark.parametrize("shape", [(6, 7), (3, 90), (2, 1300), (2, 5, 3, 3)])
def test_gradient_against_differences(shape):
    """central differences of the plain implementation, 64 bits, step 1e-4"""
    x = made(shape, torch.float32, 31, spread=1.0)
    v, i = targets_for(x, 3, 2)
    rows, vr, ir = ref.rows_of(x, 1), ref.rows_of(v, 1), ref.rows_of(i, 1).long()
    loss, dx = topk_distill_with_logits(x, v, i, 1.5, reduction="sum")
    d = ref.rows_of(dx, 1)
    for c in range(0, rows.shape[1], max(1, rows.shape[1] // 40)):
        up, down = rows.clone(), rows.clone()
        up[:, c] += 1e-4
        down[:, c] -= 1e-4
        diff = (ref.distill(up, vr, ir, 1.5, None, 1.0)[2] - ref.distill(down, vr, ir, 1.5, None, 1.0)[2]) / 2e-4
        assert (d[:, c] - diff).abs().max() < 1e-6 * (1 + diff.abs().max())


def test_upstream_gradient_scales():
    x = made((20, 50), torch.float32, 3).requires_grad_(True)
    v, i = targets_for(x.detach(), 4, 1)
    loss = topk_distill(x, v, i, 2.0)
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    (b,) = torch.autograd.grad(loss * -8.0, x)
    assert torch.equal(a * -8.0, b)            # a power of two: exact


def test_equal_calls_give_equal_bits():
    for shape in ((3000, 37), (40, 3000), (3, 100000), (2, 21, 90, 90)):
        x = made(shape, torch.bfloat16, 1)
        v, i = targets_for(x, 7, 1)
        a, b = (topk_distill_with_logits(x, v, i, 2.0) for _ in range(2))
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_on_another_stream():
    side = torch.cuda.Stream()
    x = made((64, 5000), torch.float32, 2)
    v, i = targets_for(x, 9, 1)
    want = topk_distill_with_logits(x, v, i)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = topk_distill_with_logits(x, v, i)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("shape", [(64, 40), (4, 32000), (12, 70000), (2, 21, 30, 31)])
def test_captured_and_replayed(shape):
    xs = [made(shape, torch.bfloat16, s) for s in (1, 2)]
    v, i = targets_for(xs[0], 5, 1)

    def go(leaf):
        loss = topk_distill(leaf, v, i, 2.0)
        (dx,) = torch.autograd.grad(loss, leaf)
        return [loss.detach(), dx, *topk_distill_with_logits(leaf.detach(), v, i, 2.0)]
    static = [x.clone().requires_grad_(True) for x in xs]
    go(static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(go(s))
        graphs.append(gr)
    for turn in range(3):
        fresh = [made(shape, torch.bfloat16, 10 + 2 * turn + j) for j in range(2)]
        for s, f in zip(static, fresh):
            s.data.copy_(f)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for f, o in zip(fresh, outs):
            want = go(f.clone().requires_grad_(True))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, want)), turn


@pytest.mark.parametrize("shape", [(40, 30), (20, 6000), (2, 9, 11, 13)])
def test_targets_of_a_teacher(shape):
    """the alternatives of label_log_probs as targets give the loss that the teacher's own logits give"""
    x, teacher = made(shape, torch.float32, 1), made(shape, torch.float32, 2)
    v, i = teacher_targets(teacher, 4)
    raw = teacher.gather(1, i.long())
    a, b = check(x, v, i, 2.0)[0], check(x, raw, i, 2.0)[0]
    # ln p differs from the logit by a constant per row and by its rounding: half a step of a value below 32, over T,
    # times T^2 and the |ln t - ln p| < 32 that a changed t weighs
    assert abs(a.item() - b.item()) < 2.0 ** -19 * 2 * 33
    masked = teacher.clone()
    masked[:, 3:] = -INF                                  # three classes for four places
    v, i = teacher_targets(masked, 4)
    assert (i.movedim(1, -1)[..., 3] == -1).all()
    check(x, v, i, 2.0)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_criterion(reduction):
    crit = TopKDistillLoss(2.0, reduction)
    x = made((2, 6, 9, 9), torch.float32, 1).requires_grad_(True)
    v, i = targets_for(x.detach(), 3, 1)
    w = torch.rand(2, 9, 9, generator=torch.Generator().manual_seed(1)).to(DEV)
    for t in ((v, i), (v, i, w)):
        loss = crit(x, t)
        (dx,) = torch.autograd.grad(loss, x)
        value, grad = crit.value_and_grad(x.detach(), t)
        assert torch.allclose(loss.detach(), value, rtol=1e-6) and torch.allclose(dx, grad, rtol=1e-5, atol=1e-9)


def test_light_network_learns_from_the_heavy_one():
    """the whole chain: U-Net teacher -> stored targets -> LUNeXt student through its trainer (one-pass value and gradient)
    and through autograd on the module: same loss, same logits' gradient"""
    torch.manual_seed(0)
    classes = 5
    teacher = unet_amd.UNet(3, classes).to(DEV).eval()
    student = unet_amd.LUNeXt(3, classes).to(DEV).train()
    images = torch.rand(2, 3, 32, 48, generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        targets = teacher_targets(teacher(images), 3)
    crit = TopKDistillLoss(2.0)
    import copy
    twin = copy.deepcopy(student)
    loss = crit(twin(images), targets)
    loss.backward()
    from unet_amd.dp import DataParallelTrainer, LUNeXtTrainer
    trainer = LUNeXtTrainer(student, lr=1e-3, criterion=crit, standalone=True)
    first = trainer.train_step(images, targets)
    assert torch.allclose(first, loss.detach(), rtol=1e-5), (first.item(), loss.item())
    a, b = trainer.grads.views["final_conv.weight"], twin.final_conv.weight.grad
    assert torch.allclose(a, b, rtol=1e-3, atol=1e-3 * b.abs().max().item())
    other = trainer.train_step(images, targets)
    assert torch.isfinite(other)
    # the heavy network as the student of another
    heavy = DataParallelTrainer(unet_amd.UNet(3, classes).to(DEV), criterion=crit, standalone=True)
    one = heavy.train_step(images, targets)
    assert torch.isfinite(one)
    # what the student answers, with its uncertainty
    student.eval()
    with torch.no_grad():
        lp = label_log_probs(student(images), targets[1][:, 0], top=2)
    assert lp.log_prob.shape == (2, 32, 48) and (lp.entropy >= 0).all() and (lp.top_index[:, 0] >= 0).all()


PARTS = [(1, 4097), (3, 20000), (2, 131072), (700, 70001)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", PARTS)
def test_parts_that_nobody_waits_for(shape, dtype, monkeypatch):
    """a row's parts give the same bits whether their statistics arrive or are worked out by those who need them"""
    x = made(shape, dtype, 61)
    x[0, 5] = -INF
    if shape[0] > 2:
        x[1] *= 2.0 ** 7
        x[2] = -INF
        x[2, -3:] = 1.0
    if dtype == torch.float32:
        x[-1] *= 2.0 ** 100
    v, i = targets_for(x.clamp(min=-50, max=50), 7, 61)
    if shape[0] > 2:
        i[2] = shape[1] - 1

    def run():
        leaf = x.detach().requires_grad_(True)
        loss = topk_distill(leaf, v, i, 2.0)
        (dx,) = torch.autograd.grad(loss, leaf)
        return (topk_distill(x, v, i, 2.0), loss.detach(), dx) + tuple(topk_distill_with_logits(x, v, i, 2.0))

    want = run()
    monkeypatch.setenv("UNET_AMD_DISTILL_SPINS", "0")
    for a, b in zip(run(), want):
        assert torch.equal(a.view(torch.uint8) if a.dim() else a.view(1).view(torch.uint8),
                           b.view(torch.uint8) if b.dim() else b.view(1).view(torch.uint8))


def test_two_calls_at_once():
    """the parts of two calls on two streams, side by side on the card, meet only their own"""
    xs = [made((96, 131072), torch.bfloat16, 62 + j) for j in range(2)]
    ts = [targets_for(x, 9, 62) for x in xs]
    want = [topk_distill_with_logits(x, *t) for x, t in zip(xs, ts)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(topk_distill_with_logits(xs[j], *ts[j]))
    torch.cuda.synchronize()
    for j in range(2):
        for loss, dx in got[j]:
            assert torch.equal(loss, want[j][0]) and torch.equal(dx, want[j][1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_most_classes(dtype):
    x = made((2, 1 << 20), dtype, 63)
    check(x, *targets_for(x, 64, 63), temperature=1.5, reduction="sum")


def test_rows_behind_32768():
    x = made((5, 5000), torch.bfloat16, 64)
    v, i = targets_for(x, 6, 64)
    few, dfew = topk_distill_with_logits(*(t.repeat(120, 1) for t in (x, v, i)), reduction="sum")    # enough not to be cut
    loss, dx = topk_distill_with_logits(*(t.repeat(7001, 1) for t in (x, v, i)), reduction="sum")
    assert torch.equal(dx.view(7001, 5, 5000), dfew[:5].expand(7001, 5, 5000))
    # the rows' losses, equal on both sides, summed in 64 bits and rounded once
    want = few.double().item() * 7001 / 120
    assert abs(loss.double().item() - want) <= 2.0 ** -24 * 2.01 * want


@pytest.mark.parametrize("shape,k", [((90, 15), 9), ((90, 16), 7), ((90, 16), 8), ((90, 40), 30), ((91, 64), 64), ((1, 8, 5, 9, 24), 8)])
def test_many_slots_of_short_rows(shape, k):
    """16 classes and eight slots: from there on 16 lanes take a row"""
    k = min(k, shape[-1])
    for dtype in TYPES:
        x = made(shape, dtype, 65)
        check(x, *targets_for(x, k, 65, dim=-1), temperature=1.5, reduction="sum", dim=-1)
        padded = made(shape[:-1] + (shape[-1] + 3,), dtype, 66)[..., :shape[-1]]
        check(padded, *targets_for(padded, k, 66, dim=-1), temperature=0.7, dim=-1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,k", [((1, 65, 64, 65), 5), ((2, 70, 50, 51), 64), ((3, 150, 41, 37), 4), ((5, 1001, 31, 29), 9), ((1, 80, 64, 64), 3),
                                     ((1, 81, 17, 241), 1)])
def test_many_rows_of_classes_that_lie_apart(shape, k, dtype):
    """from 4097 rows on a thread walks its row"""
    x = made(shape, dtype, 67)
    x[0, ::3, 0] = -INF
    check(x.clamp(min=-1e4), *targets_for(x, k, 67), temperature=1.7, reduction="sum")
    w = torch.rand((shape[0],) + shape[2:], generator=torch.Generator().manual_seed(68)).to(DEV)
    w[0, 2] = 0.0
    check(x.clamp(min=-1e4), *targets_for(x, k, 67), temperature=1.7, weight=w, grad_scale=3.0)


@pytest.mark.parametrize("c", [36, 37, 38, 56, 57, 64])
def test_short_rows_on_both_sides_of_28_kb(c):
    for dtype in TYPES:
        x = made((700, c), dtype, 69)
        check(x, *targets_for(x, 4, 69), temperature=2.0, reduction="sum")


def test_more_than_a_cache_holds():
    """past 256 MB the rows of a loss with a backward pass are read past the caches: the same bits as those of fewer rows"""
    x = made((550, 65536), torch.bfloat16, 70).repeat(4, 1)
    v, i = targets_for(x[:550], 5, 70)
    v, i = v.repeat(4, 1), i.repeat(4, 1)
    grads = []
    for n in (2200, 1100):
        leaf = x[:n].detach().requires_grad_(True)
        (dx,) = torch.autograd.grad(topk_distill(leaf, v[:n], i[:n], reduction="sum"), leaf)
        grads.append(dx)
    assert torch.equal(grads[0][:1100], grads[1]) and torch.equal(grads[0][1100:], grads[1])
