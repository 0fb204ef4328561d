"""The norm of a set of gradients, and clipping by it, through dg_grad_norm / dg_clip_grad_norm (gradnorm.hip): the
steps of torch.nn.utils.clip_grad_norm_ in a few launches whatever the number of tensors, with 64-bit sums in a fixed order.
SparseGaussianAdam.step(max_norm=...) clips without rewriting the gradients."""
from __future__ import annotations

import math
from array import array
from typing import Iterable

import numpy as np
import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}     # dogs_hip.h DG_F32, DG_F16, DG_BF16
_ORDERS = {2.0: 2, 1.0: 1, math.inf: 0}


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, in any order of its dimensions (channels last, transposed)."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _extent(t: torch.Tensor) -> tuple:
    """The bytes between t's first and last element."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()


def _as_numpy(t: torch.Tensor) -> np.ndarray:
    """t's addresses as an array that is never read, for np.shares_memory."""
    class Layout:
        __array_interface__ = {"version": 3, "data": (t.data_ptr(), True), "typestr": f"<u{t.element_size()}",
                               "shape": tuple(t.shape), "strides": tuple(st * t.element_size() for st in t.stride())}
    return np.asarray(Layout())


def _shares_memory(a: np.ndarray, b: np.ndarray) -> bool:
    try:
        return np.shares_memory(a, b, max_work=10_000)      # exact; the work is bounded
    except np.exceptions.TooHardError:
        return True                                          # too interleaved to tell apart


def _repeats(t: torch.Tensor) -> bool:
    """Whether two of t's elements are the same memory."""
    reach = 0
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st <= reach:
            break
        reach += st * (n - 1)
    else:
        return False       # each stride steps over all that the smaller ones reach
    a = _as_numpy(t)
    for k in range(t.dim()):     # two elements whose first difference is in dimension k
        if t.shape[k] > 1 and _shares_memory(a[(0,) * k + (slice(0, 1),)], a[(0,) * k + (slice(1, None),)]):
            return True
    return False


def _check_apart(tensors: list, gapped: list, name: str) -> None:
    """Error where a gapped tensor shares memory with itself or another: the library sees its copy only.  (Tensors
    without gaps it compares itself.)"""
    for k in gapped:
        if _repeats(tensors[k]):
            raise RuntimeError(f"{name}: a gradient's elements share memory: it cannot be scaled in place")
    gapped, reaching = set(gapped), []
    for first, end, k in sorted((*_extent(t), k) for k, t in enumerate(tensors) if t.numel()):
        reaching = [r for r in reaching if r[0] > first]
        a = _as_numpy(tensors[k]) if reaching or k in gapped else None
        for r in reaching:
            if k in gapped or r[1] in gapped:
                if r[2] is None:
                    r[2] = _as_numpy(tensors[r[1]])
                if _shares_memory(a, r[2]):
                    raise RuntimeError(f"{name}: gradients to scale overlap in memory")
        reaching.append([end, k, a])


class _Table:
    """The tensors of a call as the library takes them; keeps what it points at."""

    def __init__(self, tensors: list, name: str, in_place: bool):
        _lib.refuse_unrecorded(name, tensors)
        self.device = tensors[0].device
        self.index = index = tensors[0].get_device()
        self.keep, gapped = tensors, []
        for k, t in enumerate(tensors):
            if t.layout is not torch.strided or t.get_device() != index or index < 0 or t.dtype not in _DTYPES:
                raise RuntimeError(f"{name}: gradients must be dense float32, float16 or bfloat16 tensors on one HIP "
                                   f"device, got {t.dtype} {t.layout} on {t.device}")
            if not t.is_contiguous() and not _dense(t):
                if self.keep is tensors:
                    self.keep = list(tensors)
                self.keep[k] = t.contiguous()
                gapped.append(k)
        if in_place and gapped:
            _check_apart(tensors, gapped, name)
        self.copies = [(tensors[k], self.keep[k]) for k in gapped]
        self.n = len(tensors)
        self.lists = (array("Q", [t.data_ptr() for t in self.keep]), array("Q", [t.numel() for t in self.keep]),
                      array("B", [_DTYPES[t.dtype] for t in self.keep]))
        self.args = (self.n, *[a.buffer_info()[0] for a in self.lists])

    def write_back(self) -> None:
        for t, c in self.copies:
            t.copy_(c)


def _order(name: str, norm_type) -> int:
    order = _ORDERS.get(float(norm_type))
    if order is None:
        raise RuntimeError(f"{name}: norm_type must be 1, 2 or inf, got {norm_type}")
    return order


def _max_norm(name: str, max_norm) -> float:
    m = float(max_norm)
    if not m >= 0.0:
        raise RuntimeError(f"{name}: max_norm must not be negative, got {max_norm}")
    return m


def _scratch(L, t: _Table) -> tuple:
    nbytes = L.dg_grad_norm_scratch_bytes(t.n)
    return torch.empty(nbytes, dtype=torch.uint8, device=t.device), nbytes


def grad_norm(tensors: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of the tensors together (norm_type 2, 1 or inf), a 0-d float32 on their device.  float32,
    float16 and bfloat16 may be mixed; no tensors: 0.  Not differentiable: forward-mode tangents are refused, and so is
    torch.jit.trace."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    order = _order("grad_norm", norm_type)
    if not tensors:
        return torch.tensor(0.0)
    t = _Table(tensors, "grad_norm", in_place=False)
    L = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=t.device)
    scratch, nbytes = _scratch(L, t)
    _lib.launch(L.dg_grad_norm, t.index, *t.args, order, 0.0, norm.data_ptr(), None, scratch.data_ptr(), nbytes)
    return norm


def clip_coefficient(tensors: list, max_norm: float) -> tuple:
    """(norm, coefficient) of the tensors' 2-norm: the norm a 0-d float32, the coefficient min(1, max_norm / (norm + 1e-6)) a
    0-d float64, on the device.  For a step that scales the gradients as it reads them."""
    max_norm = _max_norm("clip_coefficient", max_norm)
    t = _Table(tensors, "clip_coefficient", in_place=False)
    L = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=t.device)
    coef = torch.empty((), dtype=torch.float64, device=t.device)
    scratch, nbytes = _scratch(L, t)
    _lib.launch(L.dg_grad_norm, t.index, *t.args, 2, max_norm, norm.data_ptr(), coef.data_ptr(), scratch.data_ptr(), nbytes)
    return norm, coef


@torch.no_grad()
def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_: scales the parameters' gradients in place by min(1, max_norm / (norm + 1e-6)) of
    the norm of them all (norm_type 2, 1 or inf) and returns that norm, a 0-d float32 on their device.  With a
    coefficient of 1 gradients keep every bit (and are not written, but for those with gaps, which are scaled in a copy and
    copied back).  Parameters without a gradient are left out, and one that is given twice counts once; gradients that share
    memory are refused.  A norm that is NaN makes every gradient NaN, an infinite one makes them 0 (NaN where they were
    infinite, and all of them with an infinite max_norm), unless error_if_nonfinite, which reads the norm back and raises."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    order, max_norm = _order("clip_grad_norm_", norm_type), _max_norm("clip_grad_norm_", max_norm)
    grads = [p.grad for p in dict.fromkeys(parameters) if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    t = _Table(grads, "clip_grad_norm_", in_place=True)
    L = _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=t.device)
    scratch, nbytes = _scratch(L, t)
    if error_if_nonfinite:
        coef = torch.empty((), dtype=torch.float64, device=t.device)
        _lib.launch(L.dg_grad_norm, t.index, *t.args, order, max_norm, norm.data_ptr(), coef.data_ptr(), scratch.data_ptr(),
                    nbytes)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"clip_grad_norm_: the norm of the gradients is {float(norm)}")
        _lib.launch(L.dg_grad_scale, t.index, *t.args, coef.data_ptr())
    else:
        _lib.launch(L.dg_clip_grad_norm, t.index, *t.args, order, max_norm, norm.data_ptr(), scratch.data_ptr(), nbytes)
    t.write_back()
    torch.autograd.graph.increment_version([g for g in grads if not g.is_inference()])
    return norm
