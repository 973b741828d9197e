"""The global gradient norm over many tensors, and clipping by it.

What a trainer does between ``backward`` and the optimizer's step (vqvae/vqgan_trainer.py:98-104 for the parameters of the
model this quantizer sits in): a few launches over all gradients of a model instead of a few per tensor, nothing copied
to the host.  GPU only.
"""
from __future__ import annotations

import array
import math
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _lib
from ._lib import NORM_1, NORM_2, NORM_INF, check
from .projection import DTYPES
from .ops import _on_device, _raw_stream, _recording, _refuse_recording, _require_cuda

#: source and result type of a tensor scaled in place, as one word of the C interface's entry
_TWICE = {dtype: code | code << 32 for dtype, code in DTYPES.items()}

_FP32_MAX = torch.finfo(torch.float32).max

_KINDS = {1.0: NORM_1, 2.0: NORM_2, math.inf: NORM_INF}


def _kind(norm_type) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type!r}")
    return kind


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    # the C interface takes fp32: a finite one beyond it would turn infinite, and NaN over an infinite norm
    return min(max_norm, _FP32_MAX) if math.isfinite(max_norm) else max_norm


def _list(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], name: str) -> List[torch.Tensor]:
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be tensors, got {type(t).__name__}")
    kinds = {(t.dtype, t.layout, t.device) for t in tensors}       # a model has a few, however many tensors it has
    for dtype, layout, _ in kinds:
        if layout is not torch.strided:
            raise TypeError(f"{name} must be dense tensors, got {layout}")
        if dtype not in DTYPES:
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {dtype}")
    devices = {device for _, _, device in kinds}
    if len(devices) > 1:
        raise ValueError(f"{name} must share one device, got {', '.join(sorted(map(str, devices)))}")
    if len(tensors) > 65536:
        raise ValueError(f"at most 65536 tensors in one call, got {len(tensors)}")
    return tensors


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one run of memory, in whatever order (a transposed or channels_last tensor does)."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _refs(srcs: Sequence[torch.Tensor], dsts: Sequence[torch.Tensor]) -> array.array:
    """The vq_tensor_ref array of the C interface: four 64-bit words an entry."""
    words: List[int] = []
    if srcs is dsts:
        for s in srcs:
            at = s.data_ptr()
            words += (at, at, s.numel(), _TWICE[s.dtype])
    else:
        for s, d in zip(srcs, dsts):
            words += (s.data_ptr(), d.data_ptr(), s.numel(), DTYPES[s.dtype] | DTYPES[d.dtype] << 32)
    return array.array("q", words)


def _same(g: torch.Tensor, o: torch.Tensor) -> bool:
    """Whether o, of g's shape, is g's own memory in g's order: scaled in place."""
    return g is o or (g.data_ptr() == o.data_ptr() and g.dtype is o.dtype and g.stride() == o.stride())


def _spans(tensors: Sequence[torch.Tensor]) -> array.array:
    """The memory of all tensors as such an array, each from its first to its last element (with the gaps between)."""
    words: List[int] = []
    for t in tensors:
        span = t.numel() and 1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
        words += (t.data_ptr(), t.data_ptr(), span, _TWICE[t.dtype])
    return array.array("q", words)


def _runs(t: torch.Tensor):
    """t's memory as ``(first byte, byte behind the last, bytes of a run, ((distance, count) of the runs' repetitions, in bytes))``."""
    size = run = t.element_size()
    dims = sorted((st * size, n) for st, n in zip(t.stride(), t.shape) if n > 1 and st > 0)
    while dims and dims[0][0] <= run:
        distance, n = dims.pop(0)
        run += distance * (n - 1)
    return t.data_ptr(), t.data_ptr() + run + sum(distance * (n - 1) for distance, n in dims), run, dims


#: steps that the search for a common element of two tensors may take: views of one tensor need one or two for each dimension
_MEET_STEPS = 4096


def _meet(a, b) -> bool:
    """Whether two tensors, as `_runs` gives them, share a byte: whether a sum of distances, each taken as often as the places of
    a's run and of b's run along it may differ, falls where the two runs touch.  True too where that takes too long to say."""
    reach = {}
    for dims, sign in ((a[3], 1), (b[3], -1)):
        for distance, n in dims:
            low, high = reach.get(distance, (0, 0))
            reach[distance] = (low, high + n - 1) if sign > 0 else (low - n + 1, high)
    levels = sorted(reach.items(), reverse=True)
    rest = [(0, 0)]                       # least and largest sum of the levels behind each
    for distance, (low, high) in reversed(levels):
        rest.append((rest[-1][0] + distance * low, rest[-1][1] + distance * high))
    rest.reverse()
    apart = b[0] - a[0]
    todo, steps = [(0, apart - a[2] + 1, apart + b[2] - 1)], 0
    while todo:
        level, least, most = todo.pop()
        if not rest[level][0] <= most or not rest[level][1] >= least:
            continue
        if level == len(levels):
            return True
        distance, (low, high) = levels[level]
        first = max(low, -((rest[level + 1][1] - least) // distance))
        last = min(high, (most - rest[level + 1][0]) // distance)
        steps += max(0, last - first + 1)
        if steps > _MEET_STEPS:
            return True
        todo += [(level + 1, least - k * distance, most - k * distance) for k in range(first, last + 1)]
    return False


def _shared(tensors: Sequence[torch.Tensor]) -> bool:
    """Whether any two tensors share memory, gaps not counted (the columns of a matrix in several tensors do not)."""
    runs = sorted(_runs(t) for t in tensors if t.numel())
    for i, a in enumerate(runs):
        for b in runs[i + 1:]:
            if b[0] >= a[1]:
                break
            if _meet(a, b):
                return True
    return False


def _refuse_overlap(refs: array.array, strided: Optional[Sequence[torch.Tensor]] = None) -> None:
    """refs: dense tensors, or the spans of `strided` ones, which are looked at closer where those overlap."""
    if _lib.load().vq_tensor_refs_overlap(refs.buffer_info()[0], len(refs) // 4) and (strided is None or _shared(strided)):
        raise ValueError("gradients that are to be scaled share memory: each element may be given once")


def grad_norm(grads: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of all tensors together, a float32 scalar on their device.

    grads: float32, bfloat16 and float16 tensors, mixed as they come, of any shape and strides, on one GPU.  norm_type: 1, 2
    or inf.  Summed in 64 bits.  NaN and infinity come through as the formula has them.  No tensor at all: 0 (on the
    host).  The same bits on every run; may be captured in a graph.  Not differentiable: tensors that require a gradient (those
    of ``create_graph=True`` do) are refused unless under ``torch.no_grad``."""
    kind = _kind(norm_type)
    grads = _list(grads, "grads")
    if _recording():
        _refuse_recording(grads, "grad_norm")
    if torch.is_grad_enabled() and True in [t.requires_grad for t in grads]:
        raise RuntimeError("grad_norm is not differentiable, and a tensor requires a gradient: detach it, or call under torch.no_grad()")
    if not grads:
        return torch.zeros(())
    _require_cuda(grads[0], "grads")
    lib = _lib.load()
    device = grads[0].device
    with _on_device(device):
        flat = [t if t.is_contiguous() or _dense(t) else t.contiguous() for t in grads]
        norm = torch.empty((), dtype=torch.float32, device=device)
        work = torch.empty(lib.vq_grad_norm_work_bytes(len(flat)), dtype=torch.uint8, device=device)
        refs = _refs(flat, flat)
        check(lib.vq_grad_norm(refs.buffer_info()[0], len(flat), kind, norm.data_ptr(), work.data_ptr(), _raw_stream(device)), "vq_grad_norm")
    return norm


def clip_grads(grads: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
               out: Union[torch.Tensor, Sequence[torch.Tensor], None] = None) -> torch.Tensor:
    """Scales the gradients by ``min(1, max_norm / (norm + 1e-6))`` and returns ``norm`` (see :func:`grad_norm`), without a
    word to the host.

    In place, or into ``out``: one tensor per gradient, of its shape and either its type or float32 (an optimizer's
    gradients beside 16-bit ones); ``grads`` are then only read.  Every result is rounded once.  An infinite norm scales by
    0 and a NaN by NaN, as the formula has it.  A tensor given twice, tensors that share elements, and expanded tensors to
    be written are refused (views of one tensor that share none, as the columns of a matrix in two halves, are fine).  As under
    ``torch.no_grad``: neither the norm nor the scaling is part of a graph of autograd.  The same bits on every run; may be
    captured in a graph."""
    kind = _kind(norm_type)
    max_norm = _max_norm(max_norm)
    grads = _list(grads, "grads")
    if out is not None:
        out = _list(out, "out")
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients but {len(out)} tensors in out")
    if _recording():
        _refuse_recording([*grads, *(out or ())], "clip_grads")
    if not grads:
        return torch.zeros(())
    written = grads if out is None else out
    dense = True
    for g, o in zip(grads, written):
        if g is not o:
            if o.shape != g.shape:
                raise ValueError(f"out has shape {tuple(o.shape)} for a gradient of shape {tuple(g.shape)}")
            if o.dtype != g.dtype and o.dtype != torch.float32:
                raise TypeError(f"out is {o.dtype} for a {g.dtype} gradient: the same type or float32")
            if o.requires_grad and o.is_leaf and torch.is_grad_enabled():
                raise ValueError("out requires a gradient itself")
        if not (g.is_contiguous() and o.is_contiguous()):
            dense = False
            if o.numel() and any(st == 0 and sz > 1 for st, sz in zip(o.stride(), o.shape)):
                raise ValueError("an expanded tensor cannot be scaled: several of its elements are one")
    if written[0].device != grads[0].device:
        raise ValueError(f"out is on {written[0].device}, the gradients on {grads[0].device}")
    if dense:
        refs = _refs(grads, written)
        _refuse_overlap(refs)
    else:
        strided = [*written, *(g for g, o in zip(grads, written) if not _same(g, o))]
        _refuse_overlap(_spans(strided), strided)
    _require_cuda(grads[0], "grads")
    device = grads[0].device
    with _on_device(device):
        dsts, back = written, ()
        if not dense:
            with torch.no_grad():
                srcs, dsts, back = _dense_pairs(grads, written)
            refs = _refs(srcs, dsts)
        lib = _lib.load()
        norm = torch.empty((), dtype=torch.float32, device=device)
        work = torch.empty(lib.vq_grad_norm_work_bytes(len(grads)), dtype=torch.uint8, device=device)
        check(lib.vq_clip_grads(refs.buffer_info()[0], len(grads), kind, max_norm, norm.data_ptr(), work.data_ptr(),
                                _raw_stream(device)), "vq_clip_grads")
        if back:
            with torch.no_grad():
                for o, c in back:
                    o.copy_(c)
        torch.autograd.graph.increment_version(dsts)
    return norm


def _dense_pairs(grads: Sequence[torch.Tensor], written: Sequence[torch.Tensor]):
    """What the kernel reads and writes: dense runs of the same element order, the tensors themselves wherever they are
    that, copies otherwise; and the copies to be brought back, as (tensor, copy)."""
    srcs, dsts, back = [], [], []
    for g, o in zip(grads, written):
        if _dense(g) and o.stride() == g.stride():
            srcs.append(g)
            dsts.append(o)
            continue
        c = g.contiguous()
        srcs.append(c)
        if o is g:
            dsts.append(c)
            back.append((o, c))
        elif o.is_contiguous():
            dsts.append(o)
        else:
            dsts.append(torch.empty(o.shape, dtype=o.dtype, device=o.device))
            back.append((o, dsts[-1]))
    return srcs, dsts, back


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` on :func:`clip_grads`: scales the ``grad`` of every parameter in place and returns
    the norm they had, both as under ``torch.no_grad``, like torch's.  Parameters without a gradient are passed over.
    ``error_if_nonfinite`` raises RuntimeError, before anything is scaled, if the norm is not finite (this is the one case that
    waits for the GPU)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    _kind(norm_type)
    _max_norm(max_norm)
    if error_if_nonfinite and grads:
        with torch.no_grad():
            norm = grad_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, "
                               "so it cannot be clipped.")
    return clip_grads(grads, max_norm, norm_type)
