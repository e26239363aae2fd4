"""Where the logits of a call over classes lie: the `uh_class_view` of a tensor and a class dimension, and the checks that
`label_log_probs` and `topk_distill` share.  A small call is bound by what Python does around its launch, so this is lean."""
import ctypes

import torch
from torch.autograd import forward_ad
from torch._C import _cuda_getCurrentRawStream as raw_stream       # current_stream() without making a Stream object

from . import _lib

DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}       # UH_F32, UH_BF16, UH_F16
INT_BYTES = {torch.int32: 4, torch.int64: 8}
byref = ctypes.byref


def _merge(sizes, strides):
    """(elements, stride) of the dimensions seen as one, or None if no single stride walks them"""
    n, step = 1, 1
    for size, stride in zip(reversed(sizes), reversed(strides)):
        if size == 1:
            continue
        if n == 1:
            step = stride
        elif stride != n * step:
            return None
        n *= size
    return n, step


def _view(t, dim):
    shape, strides = t.shape, t.stride()
    c = shape[dim]
    if dim == 1 and len(shape) == 2:
        return _lib.ClassView(shape[0], 1, strides[0], 1, strides[1] if c > 1 else 1, c, DTYPE_CODE[t.dtype])
    outer = _merge(shape[:dim], strides[:dim])
    inner = _merge(shape[dim + 1:], strides[dim + 1:])
    if outer is None or inner is None:
        return None
    return _lib.ClassView(outer[0], inner[0], outer[1], inner[1], strides[dim] if c > 1 else 1, c, DTYPE_CODE[t.dtype])


class Rows:
    """The logits of one call as rows of classes: `x` (the tensor, or a dense copy where no two strides describe it), its
    view for the kernels, the shape of what belongs to a row, and the shape of k entries per row."""
    __slots__ = ("x", "view", "rows", "classes", "row_shape", "dim", "device", "switch", "stream")

    def __init__(self, logits, dim, what):
        if not isinstance(logits, torch.Tensor) or logits.dtype not in DTYPE_CODE:
            raise ValueError(f"{what}: logits must be a fp32, bf16 or fp16 tensor")
        shape = logits.shape
        nd = len(shape)
        if nd < 1 or not -nd <= dim < nd:
            raise ValueError(f"{what}: no class dimension {dim} in logits of shape {tuple(shape)}")
        self.dim = dim = dim % nd
        self.classes = c = shape[dim]
        if not 0 < c <= _lib.CLASSES_MAX:
            raise ValueError(f"{what}: {c} classes (1 to {_lib.CLASSES_MAX})")
        self.row_shape = shape[:dim] + shape[dim + 1:]
        self.rows = logits.numel() // c
        if self.rows > 0x7fffffff:
            raise ValueError(f"{what}: {self.rows} rows (at most 2^31 - 1)")
        self.x = x = logits.detach()
        self.view = None
        if self.rows:
            self.view = _view(x, dim)
            if self.view is None:
                self.x = x = x.contiguous()
                self.view = _view(x, dim)
        self.device = logits.device

    def bind(self, what):
        """after the checks of the arguments: the stream of the launches (the tensors' device's current one)"""
        index = self.device.index
        if self.device.type != "cuda":
            raise RuntimeError(f"unet_amd.{what} runs on the HIP kernels only: tensors must be on a ROCm device")
        # a launch goes to the current device: make the tensors' own the current one around it if it is another
        self.switch = index != torch.cuda.current_device()
        self.stream = raw_stream(index)
        return self

    def new_grad(self, x):
        """an empty gradient tensor (the strides of the logits `x` where those are dense) and its view"""
        g = torch.empty_like(x)
        if g.stride() == x.stride():
            return g, self.view
        view = _view(g, self.dim)
        if view is None:
            g = torch.empty_like(x, memory_format=torch.contiguous_format)
            view = _view(g, self.dim)
        return g, view

    def entries(self, k):
        """shape of a tensor with k entries per row in the place of the classes"""
        return self.row_shape[:self.dim] + (k,) + self.row_shape[self.dim:]

    def per_row(self, t, what, dtypes):
        """a tensor with one value per row, dense in the rows' order"""
        if not isinstance(t, torch.Tensor) or t.shape != self.row_shape:
            raise ValueError(f"{what}: expected shape {tuple(self.row_shape)}, got "
                             f"{tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__}")
        return self.same_device(t, what, dtypes)

    def same_device(self, t, what, dtypes):
        if t.dtype not in dtypes:
            raise ValueError(f"{what}: dtype {t.dtype} (expected one of {', '.join(str(d) for d in dtypes)})")
        if t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the logits are on {self.device}")
        if t.requires_grad:
            t = t.detach()
        return t if t.is_contiguous() else t.contiguous()

    def call(self, name, *args):
        if self.switch:
            with torch.cuda.device(self.device):
                _lib.call(name, *args, self.stream)
        else:
            _lib.call(name, *args, self.stream)


def fp32_rows(g):
    """an upstream gradient as the kernels read it (None stays None)"""
    if g is None:
        return None
    if g.dtype is not torch.float32:
        g = g.float()
    return g if g.is_contiguous() else g.contiguous()


def refuse_tangents(what, *tensors):
    """The kernels would leave a forward-mode tangent behind without a word."""
    if forward_ad._current_level >= 0:                # inside a dual_level: outside of one there are none
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: the forward-mode gradient is not built")


def checked_temperature(temperature, what):
    t = float(temperature)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"{what}: temperature {temperature} (1e-6 to 1e6)")
    return t
