"""label_log_probs against a plain 64-bit implementation (tests/class_rows_ref.py): values, alternatives, gradients, masks,
strides, streams and graphs.  The tolerances there count the roundings of the kernels' fp32 arithmetic."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from conftest import gpu_present            # noqa: E402

if not gpu_present():
    pytest.skip("needs a GPU", allow_module_level=True)

import class_rows_ref as ref                 # noqa: E402
from unet_amd import label_log_probs         # noqa: E402

DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = math.inf, math.nan


def made(shape, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype).to(DEV)


def labels_for(logits, dim, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed + 1000)
    shape = list(logits.shape)
    c = shape.pop(dim % logits.dim())
    return torch.randint(0, c, shape, generator=g).to(dtype).to(DEV)


def check(logits, labels, top=0, temperature=1.0, dim=1, ignore_index=-100, grads=True, seed=5):
    """forward values, alternatives and gradients of one call against the plain implementation"""
    x = ref.rows_of(logits, dim)
    n, c = x.shape
    lab = None if labels is None else labels.reshape(-1).cpu().long()
    want = ref.label_probs(x, lab, top, temperature, ignore_index)
    leaf = logits.detach().requires_grad_(grads)
    got = label_log_probs(leaf, labels, top=top, temperature=temperature, dim=dim, ignore_index=ignore_index)
    flat = lambda t: t.detach().movedim(dim, -1).reshape(n, -1)                         # noqa: E731
    lt = ref.log_tol(x, c, temperature)
    ref.close(got.entropy.reshape(-1), want["entropy"], ref.entropy_tol(x, temperature), "entropy")
    if labels is None:
        assert got.log_prob is None
    else:
        assert got.log_prob.dtype == torch.float32 and got.log_prob.shape == labels.shape
        ref.close(got.log_prob.reshape(-1), want["log_prob"], lt.gather(1, lab.clamp(0, c - 1)[:, None])[:, 0], "log_prob")
    if top:
        assert got.top_index.dtype == torch.int32 and not got.top_log_prob.requires_grad
        assert torch.equal(flat(got.top_index).cpu().long(), want["index"]), "top_index"
        at = want["index"].clamp(0, c - 1)
        ref.close(flat(got.top_log_prob), want["top"], lt.gather(1, at), "top_log_prob")
    else:
        assert got.top_log_prob is None and got.top_index is None
    if grads:
        gen = torch.Generator().manual_seed(seed)
        g = torch.randn(n, generator=gen) if labels is not None else None
        h = torch.randn(n, generator=gen) * 0.3
        outs, ups = [got.entropy], [h.to(DEV).reshape(got.entropy.shape)]
        if g is not None:
            outs.append(got.log_prob)
            ups.append(g.to(DEV).reshape(got.log_prob.shape))
        (dx,) = torch.autograd.grad(outs, leaf, ups)
        assert dx.dtype == logits.dtype and dx.shape == logits.shape
        g64 = None if g is None else g.double()
        d = ref.label_probs_grad(x, lab, temperature, g64, h.double(), ignore_index)
        p = torch.nan_to_num(want["p"])
        coef = ((0 if g is None else g64.abs()) + 0 * h.double()) / temperature
        hl = (h.double().abs()[:, None] * (torch.nan_to_num(want["logp"], neginf=0.0).abs() + want["entropy"].nan_to_num()[:, None])) / temperature
        tol = ref.grad_tol(logits.dtype, d, p, coef, x, c, temperature) + torch.nan_to_num(
            p * hl * (lt + 2.0 ** -24 * 12)) + p * (h.double().abs() / temperature)[:, None] * torch.nan_to_num(
            lt + ref.entropy_tol(x, temperature)[:, None])
        ref.close(dx.detach().movedim(dim, -1).reshape(n, c), d, tol, "gradient")
    return got


ROWS = [(1, 1), (1, 2), (5, 3), (130, 7), (257, 19), (64, 64), (33, 65), (7, 100), (19, 129), (3, 511), (6, 513), (5, 1000),
        (4, 2049), (3, 4097), (2, 5003), (2, 8191), (1, 16385), (3, 32000), (2, 33001), (1, 70001), (2, 131072), (1, 140003)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,c", ROWS)
def test_rows(n, c, dtype):
    x = made((n, c), dtype, n * 7919 + c)
    check(x, labels_for(x, 1, c), top=min(c, 5), temperature=1.0)


@pytest.mark.parametrize("top", [1, 2, 3, 8, 9, 17, 33, 64])
@pytest.mark.parametrize("n,c", [(70, 64), (9, 300), (5, 2000), (4, 9001), (3, 40000), (2, 131072), (600, 70)])
def test_alternatives_of_rows(n, c, top):
    check(made((n, c), torch.bfloat16, c + top), None, top=top, temperature=2.0, grads=False)
    check(made((n, c), torch.float32, c + top), None, top=top, temperature=0.5, grads=False)


MAPS = [(1, 2, 1, 3), (2, 1, 5, 7), (1, 5, 16, 16), (3, 8, 9, 11), (2, 19, 33, 21), (1, 21, 64, 64), (2, 33, 12, 10), (1, 64, 8, 9),
        (1, 65, 16, 17), (2, 100, 7, 5), (1, 300, 4, 33), (1, 2000, 3, 5)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", MAPS)
def test_class_maps(shape, dtype):
    x = made(shape, dtype, sum(shape))
    check(x, labels_for(x, 1, 3), top=min(shape[1], 3), temperature=0.75)


@pytest.mark.parametrize("top", [1, 4, 5, 8, 9, 20, 64])
@pytest.mark.parametrize("classes", [20, 64, 70, 130])
def test_alternatives_of_class_maps(classes, top):
    if top > classes:
        pytest.skip("more alternatives than classes are refused")
    check(made((2, classes, 9, 15), torch.float32, classes * top), None, top=top, grads=False)
    check(made((2, classes, 8, 16), torch.bfloat16, classes * top), None, top=top, grads=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(40, 12), (9, 300), (5, 5000), (2, 40000), (1, 150000), (2, 12, 6, 10), (1, 90, 5, 7)])
def test_equal_logits_go_to_the_lowest_class(shape, dtype):
    """few different values; all equal; +0 beside -0"""
    c = shape[1]
    top = min(c, 64 if len(shape) == 2 else 12)
    x = made(shape, dtype, 3).mul(0.5).round()
    check(x, None, top=top, grads=False)
    check(torch.zeros(shape, dtype=dtype, device=DEV), None, top=top)
    z = torch.zeros(shape, dtype=dtype, device=DEV)
    z[:, ::2] = -0.0
    check(z, None, top=top, grads=False)


@pytest.mark.parametrize("c", [50, 700, 9000, 40000, 131072])
def test_sorted_logits(c):
    """rising and falling along the classes: the best lie side by side"""
    up = torch.linspace(-8, 8, c).expand(3, c).contiguous()
    for x in (up, up.flip(1), torch.cat([up[:, : c // 2], up[:, : c - c // 2].flip(1)], 1)):
        check(x.to(DEV), None, top=min(c, 64), grads=False)
        check(x.bfloat16().to(DEV), None, top=min(c, 64), grads=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(12, 9), (12, 64), (12, 200), (12, 1500), (12, 9000), (12, 40000), (3, 9, 2, 2), (3, 70, 2, 2)])
def test_masked_infinite_and_undefined_rows(shape, dtype):
    x = made(shape, dtype, 11)
    r = x.movedim(1, -1).reshape(-1, shape[1]).clone()
    low = torch.finfo(dtype).min
    r[0] = -INF                       # nothing left
    r[1] = low                        # masked with the type's lowest value throughout: uniform
    r[2, 1:] = -INF                   # one class left
    r[3, ::2] = -INF
    r[4, ::2] = low
    r[5, shape[1] // 2] = NAN
    r[6] = NAN
    r[7, shape[1] - 1] = INF
    r[8, :] = -INF
    r[8, 3:5] = 1.0                   # fewer classes than alternatives
    r[9, 0] = NAN
    r[10] = torch.finfo(dtype).max
    r[11, 0], r[11, 1:] = torch.finfo(dtype).max, low
    x = r.reshape(x.movedim(1, -1).shape).movedim(-1, 1).contiguous()
    lab = labels_for(x, 1, 2)
    flat = lab.reshape(-1)
    flat[2], flat[3], flat[4] = 0, 0, 0          # the class left over; masked classes as labels
    flat[11] = 0
    for t in (1.0, 0.5, 4.0):
        check(x, lab, top=min(6, shape[1]), temperature=t)
    check(x, None, top=min(64, shape[1]))


@pytest.mark.parametrize("shape", [(50, 30), (50, 500), (20, 5000), (3, 9, 5, 7)])
def test_ignored_rows_and_labels_outside_the_classes(shape):
    x = made(shape, torch.float32, 21)
    lab = labels_for(x, 1, 4)
    flat = lab.view(-1)
    flat[::3] = -100
    flat[1], flat[4] = shape[1], -7
    check(x, lab, top=3)
    lab2 = torch.where(lab == -100, 255, lab).int()
    check(x, lab2, top=2, ignore_index=255)
    # an ignored row may hold anything
    xx = x.clone()
    xx.movedim(1, -1).reshape(-1, shape[1])
    m = (lab == -100).unsqueeze(1).expand(x.shape)
    xx[m] = NAN
    check(xx, lab, top=3)


def test_every_row_ignored():
    x = made((17, 40), torch.float32, 2)
    check(x, torch.full((17,), -100, device=DEV), top=4)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides(dtype):
    """class-last images, rows inside wider buffers, odd starts, transposed, expanded and sliced logits"""
    base = made((2, 6, 10, 300), dtype, 8)
    last = base.permute(0, 3, 1, 2)                                    # [2, 300, 6, 10], classes contiguous
    check(last, labels_for(last, 1, 1), top=4)
    small = made((3, 5, 7, 11), dtype, 9).permute(0, 3, 1, 2)
    check(small, labels_for(small, 1, 1), top=4)
    for c in (21, 333, 5001):
        wide = made((9, c + 13), dtype, 10)
        for off in (0, 1, 5):
            rows = wide[:, off:off + c]
            check(rows, labels_for(rows, 1, 1), top=4)
        rows = wide[::2, 3:3 + c]
        check(rows, labels_for(rows, 1, 1), top=4)
    t = made((40, 9), dtype, 11).t()                                   # [9, 40], stride 1 between rows
    check(t, labels_for(t, 1, 1), top=4)
    e = made((1, 40), dtype, 12).expand(5, 40)
    check(e, labels_for(e, 1, 1), top=4)
    e = made((6, 1), dtype, 12).expand(6, 9)
    check(e, labels_for(e, 1, 1), top=4)
    s = made((2, 8, 9, 10), dtype, 13)[:, 1:6, 2:7, ::3]               # no two strides: copied first
    check(s, labels_for(s, 1, 1), top=3)
    seq = made((2, 3, 130), dtype, 14)
    check(seq, labels_for(seq, -1, 1), top=3, dim=-1)
    check(seq, labels_for(seq, 0, 1), top=2, dim=0)
    one = made((77,), dtype, 15)
    check(one, labels_for(one, 0, 1), top=3, dim=0)
    odd = made((2, 7, 5, 5), dtype, 16)[:, :, 1:]                      # images start inside a wider plane
    check(odd, labels_for(odd, 1, 1), top=3)


def test_no_rows_and_single_values():
    x = torch.empty(0, 5, device=DEV, requires_grad=True)
    got = label_log_probs(x, torch.empty(0, dtype=torch.int64, device=DEV), top=2)
    assert got.log_prob.shape == (0,) and got.top_index.shape == (0, 2)
    (dx,) = torch.autograd.grad(got.log_prob.sum(), x)
    assert dx.shape == x.shape


def test_offsets_past_32_bits():
    step = 1_100_000_000
    buf = torch.empty(2 * step + 2000, dtype=torch.bfloat16, device=DEV)
    rows = buf.as_strided((3, 1000), (step, 1))
    rows.copy_(made((3, 1000), torch.bfloat16, 4))
    check(rows, labels_for(rows, 1, 1), top=5, grads=False)
    maps = buf.as_strided((1, 3, 4, 30), (0, step, 30, 1))
    maps.copy_(made((1, 3, 4, 30), torch.bfloat16, 5))
    check(maps, labels_for(maps, 1, 1), top=2, grads=False)


@pytest.mark.parametrize("shape", [(6, 7), (3, 90), (2, 1300), (2, 5, 3, 3)])
def test_gradient_against_differences(shape):
    """central differences of the plain implementation, 64 bits, step 1e-4: their own error is of order 1e-8"""
    x = made(shape, torch.float32, 31, spread=1.0)
    lab = labels_for(x, 1, 6)
    rows = ref.rows_of(x, 1)
    l64 = lab.reshape(-1).cpu()
    gen = torch.Generator().manual_seed(1)
    g, h = torch.randn(len(rows), generator=gen).double(), torch.randn(len(rows), generator=gen).double()

    def value(r):
        w = ref.label_probs(r, l64, 0, 1.5)
        return g * w["log_prob"] + h * w["entropy"]
    leaf = x.requires_grad_(True)
    got = label_log_probs(leaf, lab, temperature=1.5)
    (dx,) = torch.autograd.grad((got.log_prob, got.entropy), leaf, (g.float().to(DEV).view(lab.shape), h.float().to(DEV).view(lab.shape)))
    d = ref.rows_of(dx, 1)
    for c in range(0, rows.shape[1], max(1, rows.shape[1] // 40)):
        up, down = rows.clone(), rows.clone()
        up[:, c] += 1e-4
        down[:, c] -= 1e-4
        diff = (value(up) - value(down)) / 2e-4
        assert (d[:, c] - diff).abs().max() < 1e-6 * (1 + diff.abs().max())


def test_one_gradient_of_the_two():
    x = made((11, 45), torch.float32, 5).requires_grad_(True)
    lab = labels_for(x, 1, 2)
    rows, l64 = ref.rows_of(x, 1), lab.cpu()
    got = label_log_probs(x, lab, top=3)
    (a,) = torch.autograd.grad(got.log_prob.sum(), x, retain_graph=True)
    (b,) = torch.autograd.grad(got.entropy.sum(), x)
    one = torch.ones(11, dtype=torch.float64)
    assert (ref.rows_of(a, 1) - ref.label_probs_grad(rows, l64, 1.0, one, None)).abs().max() < 1e-6
    assert (ref.rows_of(b, 1) - ref.label_probs_grad(rows, l64, 1.0, None, one)).abs().max() < 2e-6


def test_equal_calls_give_equal_bits():
    for shape in ((300, 37), (40, 3000), (3, 100000), (2, 21, 40, 40)):
        x = made(shape, torch.bfloat16, 1)
        lab = labels_for(x, 1, 1)
        a, b = (label_log_probs(x, lab, top=7) for _ in range(2))
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_on_another_stream():
    side = torch.cuda.Stream()
    x = made((64, 5000), torch.float32, 2)
    lab = labels_for(x, 1, 2)
    want = label_log_probs(x, lab, top=9)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = label_log_probs(x, lab, top=9)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("shape", [(64, 40), (4, 32000), (12, 70000), (2, 21, 30, 31)])
def test_captured_and_replayed(shape):
    """two graphs of the same call, replayed in turn with new inputs and eager work between: their workspaces are apart"""
    xs = [made(shape, torch.bfloat16, s) for s in (1, 2)]
    lab = labels_for(xs[0], 1, 1)
    ups = torch.randn(lab.shape, generator=torch.Generator().manual_seed(1)).to(DEV)

    def go(leaf):
        got = label_log_probs(leaf, lab, top=5)
        (dx,) = torch.autograd.grad((got.log_prob, got.entropy), leaf, (ups, ups))
        return [t.detach() for t in got] + [dx]
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
        fresh = [made(shape, torch.bfloat16, 10 + 2 * turn + i) for i in range(2)]
        for s, f in zip(static, fresh):
            s.data.copy_(f)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for f, o in zip(fresh, outs):
            want = go(f.clone().requires_grad_(True))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, want)), turn


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_most_classes(dtype):
    x = made((2, 1 << 20), dtype, 41)
    check(x, labels_for(x, 1, 41), top=64, temperature=0.9)
    check(x, None, grads=False)


def test_rows_behind_32768():
    """rows in parts are a launch's second dimension, and its third past 32768 of them"""
    x = made((5, 5000), torch.bfloat16, 42)
    y = labels_for(x, 1, 42)
    few = label_log_probs(x.repeat(120, 1), y.repeat(120), top=9)          # enough rows for them not to be cut
    many = label_log_probs(x.repeat(7001, 1), y.repeat(7001), top=9)
    for a, b in zip(few, many):
        assert torch.equal(b.view(7001, *a[:5].shape), a[:5].expand(7001, *a[:5].shape))


@pytest.mark.parametrize("c", [40, 300, 3000, 9000, 40000])
def test_logits_past_2_to_99(c):
    """the scale of the exponents changes at 2^100, and the running sums give way at 2^99"""
    x = made((6, c), torch.float32, 43)
    x[0] *= 2.0 ** 99
    x[1] *= 2.0 ** 102
    x[2] = x[2] - 2.0 ** 101
    x[3, c // 2] = 2.0 ** 99
    x[4, c // 3] = -2.0 ** 99
    x[5] = -x[5].abs() * 2.0 ** 120 - 2.0 ** 122
    r = label_log_probs(x, labels_for(x, 1, 43), top=4)
    want = ref.label_probs(ref.rows_of(x, 1), labels_for(x, 1, 43).cpu(), 4, 1.0)
    assert torch.equal(r.top_index.cpu().long(), want["index"])
    ref.close(r.entropy, want["entropy"], ref.entropy_tol(ref.rows_of(x, 1), 1.0), "entropy")
    ref.close(r.top_log_prob[:, 0], want["top"][:, 0], ref.log_tol(ref.rows_of(x, 1), c, 1.0).amin(1), "largest")


@pytest.mark.parametrize("temperature", [1e-6, 1e6])
@pytest.mark.parametrize("shape", [(70, 12), (20, 300), (9, 3000), (4, 40000), (1, 12, 9, 9), (2, 90, 16, 17)])
def test_widest_temperatures(shape, temperature):
    x = made(shape, torch.bfloat16, 44)
    check(x, labels_for(x, 1, 44), top=3, temperature=temperature, grads=temperature > 1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,top", [((1, 65, 64, 65), 5), ((2, 70, 50, 51), 64), ((3, 150, 41, 37), 4), ((5, 1001, 31, 29), 9), ((1, 80, 64, 64), 3),
                                       ((1, 81, 17, 241), 0)])
def test_many_rows_of_classes_that_lie_apart(shape, top, dtype):
    """from 4097 rows on a thread walks its row"""
    x = made(shape, dtype, 45)
    x[0, ::3, 0] = -INF
    x[0, :, 1] = -INF
    check(x, labels_for(x, 1, 45), top=top, temperature=1.7)


def test_more_than_a_cache_holds():
    """past 256 MB the rows of a training call are read past the caches: the same bits as those of fewer rows"""
    x = made((550, 65536), torch.bfloat16, 46).repeat(4, 1)
    y = labels_for(x, 1, 46)
    results = []
    for n in (2200, 1000):
        leaf = x[:n].detach().requires_grad_(True)
        r = label_log_probs(leaf, y[:n])
        (dx,) = torch.autograd.grad([r.log_prob.sum() + r.entropy.sum()], leaf)
        results.append((r.log_prob.detach(), r.entropy.detach(), dx))
    for a, b in zip(*results):
        assert torch.equal(a[:1000], b)
