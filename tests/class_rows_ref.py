"""Plain 64-bit implementations, on the CPU, of what tests/test_top_label_probs_gpu.py and tests/test_topk_distill_gpu.py check,
and the tolerances that follow from the kernels' arithmetic."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the distance of the smallest subnormal numbers: what a rounding to the type costs near zero
HALF_TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def rows_of(t, dim):
    """[rows, C] in 64 bits on the CPU"""
    t = t.detach().double().cpu().movedim(dim, -1)
    return t.reshape(-1, t.shape[-1])


def softmax_parts(x, temperature):
    """(log p, defined, empty) of [rows, C] 64-bit logits; undefined rows hold a NaN or +inf, empty ones only -inf"""
    defined = ~(torch.isnan(x) | (x == math.inf)).any(1)
    empty = (x == -math.inf).all(1)
    safe = torch.where((defined & ~empty)[:, None], x, torch.zeros_like(x))
    z = (safe - safe.max(1, keepdim=True).values) / temperature
    logp = z - z.exp().sum(1, keepdim=True).log()
    logp = torch.where(empty[:, None], torch.full_like(logp, -math.inf), logp)
    return torch.where(defined[:, None], logp, torch.full_like(logp, math.nan)), defined, empty


def label_probs(x, labels, top, temperature, ignore_index=-100):
    """x [rows, C] 64-bit, labels [rows] or None -> dict of 64-bit results (index: int64)"""
    n, c = x.shape
    logp, defined, empty = softmax_parts(x, temperature)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    ent = torch.where(defined, -plogp.sum(1), torch.full((n,), math.nan, dtype=torch.float64))
    ignored = torch.zeros(n, dtype=torch.bool) if labels is None else labels == ignore_index
    out = dict(entropy=torch.where(ignored, 0.0, ent), logp=logp, p=p, ignored=ignored, defined=defined, empty=empty)
    if labels is not None:
        inside = (labels >= 0) & (labels < c)
        lp = logp.gather(1, labels.clamp(0, c - 1)[:, None])[:, 0]
        lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
        out["log_prob"] = torch.where(ignored, 0.0, lp)
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        val = logp.gather(1, order)
        none = (x.gather(1, order) == -math.inf) | ignored[:, None]
        order = torch.where(none, -1, order)
        val = torch.where(none, -math.inf, val)
        out["index"] = torch.where(defined[:, None] | ignored[:, None], order, -1)
        out["top"] = torch.where(defined[:, None] | ignored[:, None], val, math.nan)
    return out


def label_probs_grad(x, labels, temperature, g, h, ignore_index=-100):
    """the formula of the gradient, [rows, C]; g, h per row or None"""
    r = label_probs(x, labels, 0, temperature, ignore_index)
    n, c = x.shape
    logp, p = r["logp"], r["p"]
    d = torch.zeros_like(x)
    if g is not None:
        hot = torch.zeros_like(x).scatter_(1, labels.clamp(0, c - 1)[:, None], 1.0)
        bad = ((labels < 0) | (labels >= c))[:, None]
        d = d + torch.where(bad, math.nan, g[:, None] * (hot - p))
    if h is not None:
        lp = torch.where(p > 0, logp, torch.zeros_like(logp))
        d = d - h[:, None] * p * (lp + r["entropy"][:, None])
    d = torch.where(r["empty"][:, None], 0.0, d / temperature)
    return torch.where(r["ignored"][:, None], 0.0, d)


def distill(x, v, idx, temperature, weight, scale):
    """(loss, d loss / dx [rows, C], per-row losses): x [rows, C], v and idx [rows, K], weight [rows] or None"""
    n, c = x.shape
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    free = idx < 0
    v = torch.where(free & ~torch.isnan(v), -math.inf, v)
    logp, _, _ = softmax_parts(x, temperature)
    off = (w == 0) | ((v == -math.inf) & (idx < c)).all(1)
    bad = (torch.isnan(v) | (idx >= c) | (v == math.inf)).any(1)
    safe = torch.where((off | bad)[:, None], torch.zeros_like(v), v)
    zv = (safe - safe.max(1, keepdim=True).values) / temperature
    logt = zv - zv.exp().sum(1, keepdim=True).log()
    t = torch.where(free, 0.0, logt.exp())
    t = torch.where(off[:, None], 0.0, t)
    at = idx.clamp(0, c - 1)
    kl = torch.where(t > 0, t * (logt - logp.gather(1, at)), torch.zeros_like(t)).sum(1)
    kl = torch.where(bad, math.nan, kl)
    rows = torch.where(off, 0.0, w * temperature ** 2 * kl)
    target = torch.zeros_like(x).scatter_add_(1, at, t)
    grad = (w * temperature * scale)[:, None] * (logp.exp() - target)
    grad = torch.where(bad[:, None], math.nan, grad)
    return rows.sum() * scale, torch.where(off[:, None], 0.0, grad), rows


def sum_error(c):
    """Relative error of s = sum of c positive terms as the kernels add them, in half steps of fp32.  An addition costs 1; a
    rescaling by 2^d 3.5 (the product 1, the exponential 2, the rounding of d 0.5: |d| 2^d < 0.6).  Counted for one term:
      a thread's row of up to 64 classes: c additions;
      16 or 64 lanes, at most 32 elements a lane in two chains, a tree of 7 additions: below 64 + 20;
      a workgroup, NV vectors of E elements a lane: NV E / 2 additions, a rescaling a vector and one for the row, a tree of 10,
        and 6 levels that join parts (4.5 each): NV (E / 2 + 3.5) + 40.5.  NV = 4: 70, NV = 8: 84 (E = 4) and 100 (E = 8, a part of
        more than 8192: c/64 + 20 >= 148), NV = 16: 128 and 160 (parts of more than 8192 and 16384: >= 148 and 276);
      a thread that walks more than 64 classes, 16 a turn: 16 + c/16 and 3.5 for each turn that raises its maximum, which may be
        more than the number returned; the smaller one is asked of it all the same (roundings do not all point one way)."""
    return min(c, max(-(-c // 64), 64)) + 20


def z_error(x, temperature):
    """Absolute error of z = (x - m)/T and of ln p, per row, from the roundings of the difference, of the product with (or
    division by) T, of 1/T and of T itself, in 64-bit numbers; the exponent of a term of s has the same error, weighted by the
    term, so that |z| e^z <= 1/e of it enters: counted once more."""
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    top = finite.max(1).values
    span = (torch.where(torch.isfinite(x), top[:, None] - x, torch.zeros_like(x)) / temperature).abs()
    return span, 2.0 ** -24 * 5.0


def close(got, want, tol, what):
    # a value past the type's largest rounds to infinity (masks of the type's lowest value give ln p of twice that)
    past = want.double().to(got.dtype) if got.dtype != torch.float64 else want
    got = got.detach().double().cpu()
    want = want.double()
    want = torch.where(torch.isinf(past), past.double(), want)
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} against {tuple(want.shape)}"
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    err = torch.where(same, torch.zeros_like(want), (got - want).abs())
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    bad = ~(err <= tol) & ~same
    if bad.any():
        i = bad.nonzero()[0].tolist()
        at = tuple(i)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values, first at {at}: got {got[at].item()!r}, want "
                             f"{want[at].item()!r}, tolerance {tol[at].item():.3g}")


def log_tol(x, c, temperature):
    """tolerance of ln p per element: z and ln s; a masked class has none"""
    span, e = z_error(x, temperature)
    # ln s: relative error of s, the logarithm itself (two half steps of a value up to ln c), terms' exponents (2^z within
    # two half steps, argument error weighted: below one) ; final subtraction: one half step of the result
    base = 2.0 ** -24 * (sum_error(c) + 4 + 4 * math.log(c + 1) + 4)
    return span * (e + 2.0 ** -24) + base


def grad_tol(dtype, want, p, scale_abs, x, c, temperature):
    """d = p * coef (+ own): p's relative error is that of ln p; then two products, an addition and the rounding to the
    type; scale_abs: |coef| per row"""
    lt = log_tol(x, c, temperature)
    rel = lt + 2.0 ** -24 * 8
    fp32 = torch.where(p > 0, p * rel, torch.zeros_like(p)) * scale_abs[:, None]
    fp32 = torch.nan_to_num(fp32) + 2.0 ** -24 * 4 * torch.nan_to_num(want).abs()
    # products below the smallest normal fp32 number are flushed
    return fp32 * 1.01 + HALF_STEP[dtype] * 1.01 * torch.nan_to_num(want).abs() + HALF_TINY[dtype] + 2.0 ** -125 * (
        1 + scale_abs[:, None])


def entropy_tol(x, temperature):
    """ln s as above; t = sum e^z z: its terms carry the error of their exponent, four half steps of their own and those of
    the sum, all relative to sum p |z|"""
    c = x.shape[1]
    span, e = z_error(x, temperature)
    logp, _, _ = softmax_parts(x, temperature)
    p = torch.nan_to_num(logp.exp())
    span = torch.where(p > 0, span, torch.zeros_like(span))
    spread = (p * span * (e * span + 2.0 ** -24 * (8 + sum_error(c)))).sum(1)
    return spread + 2.0 ** -24 * (sum_error(c) + 8 + 5 * math.log(c + 1))


def distill_tols(x, v, idx, temperature, weight, scale, want_grad, dtype):
    """(tolerance of the loss, tolerance of the gradient): ln t and ln p as ln p above, t relative to itself, the slots'
    sum (tree or sequence: at most K additions) and the rows' sums in 64 bits over values rounded to fp32 once"""
    n, c = x.shape
    k = v.shape[1]
    eps = 2.0 ** -24
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double().abs()
    vv = torch.where(idx < 0, -math.inf, v)
    usable = torch.isfinite(vv)
    lt = torch.where(usable, log_tol(vv, k, temperature), torch.zeros_like(vv))
    lp_all = log_tol(x, c, temperature)
    at = idx.clamp(0, c - 1)
    lp = torch.where(usable, lp_all.gather(1, at), torch.zeros_like(vv))
    logt, _, _ = softmax_parts(vv, temperature)
    t = torch.nan_to_num(logt.exp())
    logp, _, _ = softmax_parts(x, temperature)
    diff = torch.where(t > 0, logt - logp.gather(1, at), torch.zeros_like(t)).abs()
    diff = torch.nan_to_num(diff, posinf=0.0)
    row = (t * (lt + lp + diff * (lt + eps * (k + 16)))).sum(1) * temperature ** 2 * w
    loss_tol = torch.nan_to_num(row).sum() * scale * 1.01 + eps * 4
    p = torch.nan_to_num(logp.exp())
    target = torch.zeros_like(x).scatter_add_(1, at, torch.nan_to_num(t * (lt + eps * (k + 8))))
    coef = (w * temperature * scale)[:, None]
    plain = torch.zeros_like(x).scatter_add_(1, at, t)
    fp32 = coef * (torch.nan_to_num(p * (lp_all + 8 * eps)) + target + eps * 4 * (p + plain))
    grad_tol_ = fp32 * 1.01 + HALF_STEP[dtype] * 1.01 * torch.nan_to_num(want_grad).abs() + HALF_TINY[dtype] + 2.0 ** -125 * (
        1 + coef)
    return loss_tol, grad_tol_
