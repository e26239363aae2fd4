"""What is measured of the operators over class logits: `label_log_probs` (log probabilities of given labels, entropy,
top alternatives; with gradients) and `topk_distill` (distillation from a teacher's top logits; value and gradient).

A row is one prediction over C classes: a token of a batch of sequences ([rows, C]) or a pixel of a batch of class maps
([B, C, H, W], the class dimension in front of the image).  With x its logits and T the temperature,

    z = (x - max x) / T,   s = sum e^z,   p = e^z / s
    log_prob = z[label] - ln s,   entropy = ln s - (sum e^z z) / s,   top: the largest logits, ties to the lowest class
    loss = mean over rows of w T^2 sum_k t_k (ln t_k - ln p[i_k]),   t = softmax of the teacher's slots over T
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100
DIM = 1                     # the class dimension of both layouts


# ---- cases ----------------------------------------------------------------------------------------------------------
def _rows(name, op, way, rows, classes, dtype, top, temperature=1.0, **more):
    case = dict(op=op, way=way, layout="rows", batch=1, height=rows, width=1, classes=classes, dtype=dtype, top=top,
                temperature=temperature, padded=False, row_step=classes)
    case.update(more)
    if name:
        case["name"] = name
    return case


def _maps(name, op, way, batch, classes, height, width, dtype, top, temperature=1.0, **more):
    case = dict(op=op, way=way, layout="maps", batch=batch, height=height, width=width, classes=classes, dtype=dtype,
                top=top, temperature=temperature, padded=False, row_step=classes)
    case.update(more)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one step of sampling for a few sequences: the log probability of what was drawn, and its alternatives
        _rows("logprobs_few_rows", "logprobs", "forward", 4, 32000, "bf16", 20),
        # scoring a batch of texts under a vocabulary of odd size, eight alternatives for each token
        _rows("logprobs_rows_odd", "logprobs", "forward", 2047, 50021, "bf16", 8),
        # a teacher's targets under a large vocabulary: its 64 best classes for each token
        _rows("logprobs_long_rows", "logprobs", "forward", 1024, 131072, "bf16", 64),
        # training on log probabilities with an entropy term; a tenth of the tokens is padding
        _rows("logprobs_rows_train", "logprobs", "train", 4096, 32000, "bf16", 0, padded=True),
        # evaluation of class maps at the benchmark's batch and image size, with three candidates for each pixel
        _maps("logprobs_maps", "logprobs", "forward", 32, 21, 256, 256, "fp32", 3),
        # cross entropy and entropy of class maps whose planes are no multiple of a vector, with unlabelled pixels
        _maps("logprobs_maps_train", "logprobs", "train", 8, 19, 251, 333, "fp32", 0, padded=True),
        # a training step's loss on a small classification batch
        _rows("distill_few_rows", "distill", "step", 32, 1000, "fp32", 8, 4.0),
        # a training step's loss and gradient over a middle-sized vocabulary
        _rows("distill_rows", "distill", "step", 4096, 32000, "bf16", 64, 2.0),
        # the same through autograd: odd sizes, rows inside a wider buffer, padded tokens with weight zero
        _rows("distill_rows_autograd", "distill", "train", 1021, 50021, "fp16", 50, 1.0, padded=True, row_step=50176),
        # a large vocabulary: the largest call
        _rows("distill_long_rows", "distill", "step", 2048, 131072, "bf16", 100, 1.0),
        # a light segmentation network taught by a heavy one: class maps at the benchmark's batch and image size
        _maps("distill_maps", "distill", "step", 32, 21, 256, 256, "fp32", 4, 2.0),
        # the validation loss of the same, on class-last pixels
        _rows("distill_pixels", "distill", "forward", 16 * 256 * 256, 12, "bf16", 3, 2.0),
    ]


MOST_ELEMENTS = {"fp32": 1 << 26, "bf16": 1 << 27, "fp16": 1 << 27}


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("logprobs", "distill"))
    way = rng.choice(("forward", "train") if op == "logprobs" else ("forward", "train", "step"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    temperature = rng.choice((0.7, 1.0, 2.0, 4.0))
    padded = rng.random() < 0.5
    most = MOST_ELEMENTS[dtype]
    if rng.random() < 0.65:
        classes = _log_between(rng, 2, 150000)
        rows = _log_between(rng, 1, max(1, min(1 << 20, most // (classes + 16))))
        step = classes + (rng.choice((0, 0, 1, 8, 13)))
        top = _log_between(rng, 1, min(64, classes))
        if op == "logprobs" and rng.random() < 0.3:
            top = 0
        return _rows(None, op, way, rows, classes, dtype, top, temperature, padded=padded, row_step=step)
    classes = _log_between(rng, 2, 160)
    batch = _log_between(rng, 1, 32)
    height = _log_between(rng, 16, 512)
    width = _log_between(rng, 16, 512)
    while batch * classes * height * width > most:
        batch, height = max(1, batch // 2), max(16, height // 2 + 1)
        if batch == 1 and height <= 17:
            width = max(16, width // 2)
    top = _log_between(rng, 1, min(8, classes))
    if op == "logprobs" and rng.random() < 0.3:
        top = 0
    return _maps(None, op, way, batch, classes, height, width, dtype, top, temperature, padded=padded)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _shape(case, classes):
    """the tensor's shape with `classes` in the class dimension"""
    if case["layout"] == "rows":
        return (case["height"], classes)
    return (case["batch"], classes, case["height"], case["width"])


def _scale(case):
    """The loss scale that a training loop over fp16 logits keeps, so that the gradients stay inside the type."""
    rows = case["batch"] * case["height"] * case["width"]
    return float(2 ** min(16, 5 + int(math.log2(rows)))) if case["dtype"] == "fp16" else 1.0


def _inputs(case, seed):
    """Logits as a network's head gives them: a spread of a few units over the classes, one class standing out in most
    rows.  The teacher is the same signal with another noise, so that both mostly agree."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    c, dtype, dim = case["classes"], DTYPES[case["dtype"]], DIM
    rows_shape = _shape(case, 1)
    label = torch.randint(0, c, rows_shape, generator=g, device=dev)
    lift = 2.0 + 6.0 * torch.rand(rows_shape, generator=g, device=dev)
    noise = torch.randn(_shape(case, c), generator=g, device=dev).mul_(2.0)
    student = noise.scatter_add(dim, label, lift)
    if case["layout"] == "rows" and case["row_step"] > c:
        wide = torch.zeros(case["height"], case["row_step"], dtype=dtype, device=dev)
        wide[:, :c] = student
        logits = wide[:, :c]
    else:
        logits = student.to(dtype)
    labels = label.squeeze(dim)
    out = dict(logits=logits, labels=labels)
    rows = labels.shape
    if case["op"] == "logprobs":
        if case["padded"]:
            labels.masked_fill_(torch.rand(rows, generator=g, device=dev) < 0.1, IGNORE)
        if case["way"] == "train":
            n = labels.numel()
            out["grad_log_prob"] = torch.randn(rows, generator=g, device=dev).mul_(_scale(case) / n)
            out["grad_entropy"] = torch.randn(rows, generator=g, device=dev).mul_(0.01 * _scale(case) / n)
    else:
        noise.mul_(0.8).add_(torch.randn(noise.shape, generator=g, device=dev)).scatter_add_(dim, label, lift)
        value, index = torch.topk(noise, case["top"], dim=dim)
        out["top_logits"], out["top_index"] = value.to(dtype).contiguous(), index.to(torch.int32).contiguous()
        if case["padded"]:
            out["weight"] = (torch.rand(rows, generator=g, device=dev) >= 0.1).float()
        if case["way"] == "train":
            out["scale"] = torch.full((), _scale(case), device=dev)
    return out


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["way"] == "train":
        state["logits"].requires_grad_(True)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import unet_amd

    case, x = state["case"], state["logits"]
    if case["op"] == "logprobs":
        got = unet_amd.label_log_probs(x, state["labels"], top=case["top"], temperature=case["temperature"], dim=DIM,
                                       ignore_index=IGNORE)
        out = dict(log_prob=got.log_prob.detach(), entropy=got.entropy.detach())
        if case["top"]:
            out.update(top_log_prob=got.top_log_prob, top_index=got.top_index)
        if case["way"] == "train":
            (out["grad"],) = torch.autograd.grad((got.log_prob, got.entropy), x,
                                                 (state["grad_log_prob"], state["grad_entropy"]))
        return out
    if case["way"] == "step":
        loss, grad = unet_amd.topk_distill_with_logits(x, state["top_logits"], state["top_index"],
                                                       temperature=case["temperature"], weight=state.get("weight"),
                                                       grad_scale=_scale(case), dim=DIM)
        return dict(loss=loss, grad=grad)
    loss = unet_amd.topk_distill(x, state["top_logits"], state["top_index"], temperature=case["temperature"],
                                 weight=state.get("weight"), dim=DIM)
    if case["way"] == "forward":
        return dict(loss=loss)
    (grad,) = torch.autograd.grad(loss, x, state["scale"])
    return dict(loss=loss.detach(), grad=grad)


def _order_key(x, dim):
    """int64 keys whose descending order is that of the fp32 values, equal values by the lowest position"""
    bits = (x + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    shape = [1] * x.dim()
    shape[dim] = x.shape[dim]
    return key + (0x7FFFFFFF - torch.arange(x.shape[dim], device=x.device)).view(shape)


def _run_plain(state):
    case, dim = state["case"], DIM
    t = case["temperature"]
    x = state["logits"].float()
    z = (x - x.amax(dim, keepdim=True)) / t
    e = z.exp()
    s = e.sum(dim, keepdim=True)
    log_s = s.log()
    if case["op"] == "logprobs":
        labels = state["labels"].unsqueeze(dim)
        used = labels != IGNORE
        label = labels.clamp_min(0)
        log_prob = torch.where(used, z.gather(dim, label) - log_s, 0.0)
        entropy = torch.where(used, log_s - (e * z).sum(dim, keepdim=True) / s, 0.0)
        out = dict(log_prob=log_prob.squeeze(dim), entropy=entropy.squeeze(dim))
        if case["top"]:
            index = torch.topk(_order_key(x.contiguous(), dim), case["top"], dim=dim).indices
            out["top_log_prob"] = torch.where(used, z.gather(dim, index) - log_s, -math.inf)
            out["top_index"] = torch.where(used, index, -1).to(torch.int32)
        if case["way"] == "train":
            g = torch.where(used, state["grad_log_prob"].unsqueeze(dim), 0.0)
            h = torch.where(used, state["grad_entropy"].unsqueeze(dim), 0.0)
            grad = (e / s) * (-g - h * (z - log_s + entropy))
            grad.scatter_add_(dim, label, g)
            out["grad"] = (grad / t).to(state["logits"].dtype)
        return out
    v = state["top_logits"].float() / t
    index = state["top_index"].long()
    v = v - v.amax(dim, keepdim=True)
    ev = v.exp()
    sv = ev.sum(dim, keepdim=True)
    p = ev / sv
    rows = x.numel() // case["classes"]
    w = state["weight"].unsqueeze(dim) / rows if "weight" in state else torch.full_like(s, 1.0 / rows)
    per_row = (p * (v - sv.log() - (z.gather(dim, index) - log_s))).sum(dim, keepdim=True)
    out = dict(loss=(per_row.double() * w).sum().mul(t * t).float())
    if case["way"] != "forward":
        grad = e / s
        grad.scatter_add_(dim, index, -p)
        out["grad"] = (grad * (w * (t * _scale(case)))).to(state["logits"].dtype)
    return out


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    """row by row blocks in 64 bits, classes in the last dimension, laid back afterwards"""
    given = _inputs(case, seed)
    dim, t = DIM, case["temperature"]
    logits = given["logits"].movedim(dim, -1)
    rows_shape = logits.shape[:-1]
    c = case["classes"]
    x = logits.reshape(-1, c)
    n = x.shape[0]
    block = max(1, (1 << 25) // c)

    def back(rows):
        """[n, k] -> the operator's layout"""
        return rows.reshape(*rows_shape, rows.shape[-1]).movedim(-1, dim)

    parts = {}

    def keep(**outs):
        for name, value in outs.items():
            parts.setdefault(name, []).append(value)

    loss = 0.0
    for lo in range(0, n, block):
        xb = x[lo:lo + block].double() / t
        logp = xb - torch.logsumexp(xb, dim=1, keepdim=True)
        p = torch.exp(logp)
        if case["op"] == "logprobs":
            lab = given["labels"].reshape(-1)[lo:lo + block]
            on = (lab != IGNORE).double()
            safe = lab * (lab != IGNORE)
            ent = -(p * logp).sum(1)
            keep(log_prob=logp[torch.arange(len(lab), device=lab.device), safe] * on, entropy=ent * on)
            if case["top"]:
                # stable: equal logits keep the order of their classes
                order = torch.sort(x[lo:lo + block].float(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
                best = torch.gather(logp, 1, order)
                off = on[:, None] == 0
                keep(top_log_prob=best.masked_fill(off, -math.inf), top_index=order.masked_fill(off, -1).int())
            if case["way"] == "train":
                g = given["grad_log_prob"].reshape(-1)[lo:lo + block].double() * on
                h = given["grad_entropy"].reshape(-1)[lo:lo + block].double() * on
                one = torch.zeros_like(p)
                one[torch.arange(len(lab), device=lab.device), safe] = 1.0
                keep(grad=(g[:, None] * (one - p) - h[:, None] * p * (logp + ent[:, None])) / t)
        else:
            k = case["top"]
            v = given["top_logits"].movedim(dim, -1).reshape(-1, k)[lo:lo + block].double() / t
            idx = given["top_index"].movedim(dim, -1).reshape(-1, k)[lo:lo + block].long()
            logt = v - torch.logsumexp(v, dim=1, keepdim=True)
            q = torch.exp(logt)
            w = torch.ones(len(xb), dtype=torch.float64, device=xb.device)
            if "weight" in given:
                w = given["weight"].reshape(-1)[lo:lo + block].double()
            kl = (q * (logt - torch.gather(logp, 1, idx))).sum(1)
            loss = loss + (w * kl).sum() * (t * t / n)
            if case["way"] != "forward":
                target = torch.zeros_like(p).scatter_add_(1, idx, q)
                keep(grad=(p - target) * (w * (t / n * _scale(case)))[:, None])
    out = {}
    if case["op"] == "logprobs":
        out = {name: torch.cat(parts[name]).reshape(rows_shape) for name in ("log_prob", "entropy")}
        if case["top"]:
            out["top_log_prob"] = back(torch.cat(parts["top_log_prob"]))
            out["top_index"] = back(torch.cat(parts["top_index"]))
    else:
        out["loss"] = loss
    if "grad" in parts:
        out["grad"] = back(torch.cat(parts["grad"]))
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    rows = case["batch"] * case["height"] * case["width"]
    elements = rows * case["classes"]
    moved = elements * size
    if case["op"] == "logprobs":
        moved += rows * (8 + 4 + 4) + rows * case["top"] * 8
        if case["way"] == "train":
            moved += elements * size + rows * 8
    else:
        moved += rows * case["top"] * (size + 4) + 4 + (rows * 4 if case["padded"] else 0)
        if case["way"] != "forward":
            moved += elements * size
    each = 8 if case["way"] == "forward" else 14
    return {"bytes": moved, "flops": elements * each}
