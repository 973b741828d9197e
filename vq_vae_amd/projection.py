"""Linear layers with bias, activation and residual in one kernel, with their gradients.

The quantizer sits between two projections (vqvae/custom_vqgan.py:50-51); a model over its codes consists of them.
``linear`` computes ``act(x W^T + b) + residual`` on the matrix cores in fp32, bf16 or fp16: sums in fp32, one rounding
per output, no tensor in between.  For one to sixteen rows (a token, a few sequences answered together) a kernel bound by
reading the weights takes over.  GPU only, like everything here: there is no fallback.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
import torch.nn as nn

from . import _lib
from ._lib import ACTIVATIONS, LINEAR_BACKWARD, LINEAR_FORWARD, check
from .ops import _on_device, _raw_stream, _recording, _refuse_recording, _require_cuda

DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}

#: the widest distance between two rows that the kernels address (bytes)
_MAX_PITCH = 0x7fffffff // 256 - 128

_MAX_FEATURES = 1 << 20


@functools.lru_cache(maxsize=4096)
def _work_bytes(which: int, M: int, K: int, N: int, dtype: int) -> int:
    return _lib.load().vq_linear_work_bytes(which, M, K, N, dtype)


def _work(which: int, M: int, K: int, N: int, dtype: int, device) -> Optional[torch.Tensor]:
    """Scratch of one call, out of torch's allocator: calls on different streams or in different graphs never share it."""
    n = _work_bytes(which, M, K, N, dtype)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _kept(dtype: torch.dtype, activation: str) -> torch.dtype:
    """As what ``input @ weight.T + bias`` is kept for the gradient: fp16 is eight times as exact as bf16 where it matters."""
    return torch.float16 if dtype is torch.bfloat16 and activation not in ("none", "relu") else dtype


def _matrix(t: torch.Tensor, width: int):
    """t as rows of ``width`` elements, dense each and at any distance from each other: ``(a tensor that starts where they do, how
    many, elements between them)``; copied only if it is not such."""
    if t.is_contiguous():
        return t, t.numel() // width, width
    t = t if t.dim() == 2 else t.reshape(-1, width)
    rows, pitch = t.shape[0], t.stride(0)
    if (t.stride(1) == 1 or width == 1) and (rows <= 1 or width <= pitch <= _MAX_PITCH // t.element_size()):
        return t, rows, pitch if rows > 1 else width
    return t.contiguous(), rows, width


def _check(x, weight, bias, activation, residual) -> None:
    # what nearly every call passes in a third of the time of the tests below, which say what is wrong with the others
    if (isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor) and x.is_cuda and activation in ACTIVATIONS
            and weight.dim() == 2 and x.dim() > 0):
        dtype, device, (N, K), shape = x.dtype, x.get_device(), weight.shape, x.shape
        if (dtype in DTYPES and weight.dtype is dtype and weight.get_device() == device and shape[-1] == K and 0 < K <= _MAX_FEATURES
                and 0 < N <= _MAX_FEATURES
                and (bias is None or (isinstance(bias, torch.Tensor) and bias.dtype is dtype and bias.get_device() == device
                                      and bias.shape == (N,)))
                and (residual is None or (isinstance(residual, torch.Tensor) and residual.dtype is dtype
                                          and residual.get_device() == device and residual.shape == (*shape[:-1], N)))):
            return
    for t, name, optional in ((x, "input", False), (weight, "weight", False), (bias, "bias", True), (residual, "residual", True)):
        if t is None and optional:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, the input {x.dtype}: all tensors of a linear layer share one type")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, the input on {x.device}")
    if x.dtype not in DTYPES:
        raise TypeError(f"linear takes float32, bfloat16 or float16 tensors, got {x.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be (out features, in features), both at least 1, got {tuple(weight.shape)}")
    N, K = weight.shape
    if max(N, K) > _MAX_FEATURES:
        raise ValueError(f"linear takes up to {_MAX_FEATURES} features, got {tuple(weight.shape)}")
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"input {tuple(x.shape)} does not end in the weight's {K} in features")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias must have shape ({N},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        raise ValueError(f"residual must have the output's shape {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    _require_cuda(x, "input")


def linear_forward(x, weight, bias=None, activation: str = "none", residual=None, want_pre: bool = False):
    """``(y, pre)``: ``pre = x W^T + bias`` (None unless wanted) and ``y = act(pre) + residual``, without autograd.
    Arguments as :func:`linear`, already checked."""
    device = x.device
    with _on_device(device):
        K = weight.shape[1]
        return _forward(_matrix(x, K), _matrix(weight, K), K, x.shape, bias, activation, residual, want_pre, device)


def _forward(x2, w2, K: int, shape, bias, activation: str, residual, want_pre: bool, device):
    # on the current device; x2, w2: as _matrix returns them
    (x2, M, ldx), (w2, N, ldw) = x2, w2
    dt = DTYPES[x2.dtype]
    y = x2.new_empty((*shape[:-1], N))
    pre = y.new_empty(y.shape, dtype=_kept(y.dtype, activation)) if want_pre else None
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    r2, ldr = None, 0
    if residual is not None:
        r2, _, ldr = _matrix(residual, N)
    work = _work(LINEAR_FORWARD, M, K, N, dt, device)
    check(_lib.load().vq_linear(x2.data_ptr(), ldx, w2.data_ptr(), ldw, _address(b), _address(r2), ldr, dt, ACTIVATIONS[activation], M, K,
                                N, y.data_ptr(), _address(pre), _address(work), _raw_stream(device)), "vq_linear")
    return y, pre


def linear_backward(grad, x, weight, pre, activation: str, want_x: bool, want_weight: bool, want_bias: bool):
    """Gradients ``(input, weight, bias)`` of ``act(x W^T + b)`` for the output gradient ``grad`` (None where not
    wanted); ``pre`` is what :func:`linear_forward` returned (None for activation "none")."""
    with _on_device(x.device):
        K = weight.shape[1]
        x2, w2 = _matrix(x, K), _matrix(weight, K)
        p = None if pre is None else pre.contiguous()
        return _backward(_facts(x2, w2, K, activation), grad.contiguous(), x.shape, x2[0], w2[0], p, want_x, want_weight, want_bias)


def _facts(x2, w2, K: int, activation: str):
    """What a backward pass needs besides addresses."""
    (x2, M, ldx), (_, N, ldw), dt = x2, w2, DTYPES[x2[0].dtype]
    return M, K, N, dt, ACTIVATIONS[activation], ldx, ldw, _work_bytes(LINEAR_BACKWARD, M, K, N, dt)


def _backward(facts, grad, shape, x2, w2, pre, want_x: bool, want_weight: bool, want_bias: bool):
    # on the current device; x2, w2: tensors that start where the rows do; grad, pre: dense
    M, K, N, dt, act, ldx, ldw, work_bytes = facts
    device = grad.device
    gx = grad.new_empty(shape) if want_x else None
    gw = grad.new_empty((N, K)) if want_weight else None
    gb = grad.new_empty((N,)) if want_bias else None
    work = torch.empty(work_bytes, dtype=torch.uint8, device=device) if work_bytes else None
    check(_lib.load().vq_linear_backward(grad.data_ptr(), None if pre is None else pre.data_ptr(), x2.data_ptr(), ldx, w2.data_ptr(),
                                         ldw, dt, act, M, K, N, gx.data_ptr() if want_x and M else None,
                                         gw.data_ptr() if want_weight else None, gb.data_ptr() if want_bias else None,
                                         None if work is None else work.data_ptr(), _raw_stream(device)), "vq_linear_backward")
    return gx, gw, gb


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        K = weight.shape[1]
        want_pre = activation != "none" and any(ctx.needs_input_grad[:3])
        device = x.device
        with _on_device(device):
            x2, w2 = _matrix(x, K), _matrix(weight, K)
            y, pre = _forward(x2, w2, K, x.shape, bias, activation, residual, want_pre, device)
        # a backward pass on the engine's thread takes about twice as long per line as here: what it can know is found out now
        ctx.facts = _facts(x2, w2, K, activation)
        ctx.in_place = x2[0].data_ptr() == x.data_ptr() and w2[0] is weight      # the rows are the tensors' own memory
        ctx.layout = x.shape, x.stride(), weight.shape, weight.stride(), x.dtype, x.device
        ctx.activation = activation
        ctx.save_for_backward(x, weight, pre)
        return y

    @staticmethod
    def backward(ctx, grad):
        if _recording():
            _refuse_recording([grad], "the gradient of linear")
        # under create_graph the result has to refuse a second derivative; the wrapper that sees to it takes 5 us
        return _gradients_once(ctx, grad) if torch.is_grad_enabled() else _gradients(ctx, grad)


def _gradients(ctx, grad):
    x, weight, pre = ctx.saved_tensors
    want_x, want_weight, want_bias, want_residual, _ = ctx.needs_input_grad
    gx = gw = gb = None
    if want_x or want_weight or want_bias:
        # hooks on saved tensors may hand back others than were saved: other strides are fine, nothing else is
        x_shape, x_stride, w_shape, w_stride, dtype, device = ctx.layout
        if not (x.shape == x_shape and x.dtype is dtype and x.device == device
                and weight.shape == w_shape and weight.dtype is dtype and weight.device == device
                and (pre is None or (pre.shape == grad.shape and pre.dtype is _kept(dtype, ctx.activation) and pre.device == device))):
            raise RuntimeError("a hook on saved tensors returned a tensor of another shape, type or device than was saved")
        if (ctx.in_place and x.stride() == x_stride and weight.stride() == w_stride and grad.is_contiguous()
                and (pre is None or pre.is_contiguous())):
            with _on_device(device):
                gx, gw, gb = _backward(ctx.facts, grad, x_shape, x, weight, pre, want_x, want_weight, want_bias)
        else:
            gx, gw, gb = linear_backward(grad, x, weight, pre, ctx.activation, want_x, want_weight, want_bias)
    return gx, gw, gb, grad if want_residual else None, None


_gradients_once = torch.autograd.function.once_differentiable(_gradients)


def linear(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(input @ weight.T + bias) + residual``.

    input: (..., K); weight: (N, K); bias: (N,) or None; residual: (..., N) or None; the result is (..., N), dense.  One
    element type for all of them: float32, bfloat16 or float16.  activation: "none", "relu", "silu", "gelu" (the exact
    one, by the normal distribution function) or "gelu_tanh".  Rows at any distance from each other are read in place;
    other strides are copied first.  Sums are fp32 and every output is rounded once; the result is the same bits on
    every run.

    Differentiable once in all four tensors.  For an activation the forward keeps ``input @ weight.T + bias`` in fp32 or
    fp16 (bf16 layers too, but for relu), and the backward rounds the gradient behind the activation to it before the two products (the bias
    gradient is summed before that rounding).
    Forward-mode derivatives, transforms of ``torch.func`` and traces (``torch.jit.trace``, ``make_fx``) are refused.
    Under autocast the tensors keep their types, and all have to share one there too.  May be captured in a graph, backward
    included (drop every eager autograd graph over the same leaves before capturing, as torch asks for any backward under
    capture)."""
    if _recording():
        _refuse_recording((input, weight, bias, residual), "linear")
    _check(input, weight, bias, activation, residual)
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LinearFn.apply(input, weight, bias, residual, activation)
    return linear_forward(input, weight, bias, activation, residual)[0]


class Linear(nn.Linear):
    """``nn.Linear`` (same parameters, initialisation and state dict) on :func:`linear`, with the activation and an optional
    residual in the same kernel: ``layer(x, residual)`` is ``act(x W^T + b) + residual``.

    Autocast does not reach it: with fp32 parameters it refuses the 16-bit input that ``nn.Linear`` would take there.  Put the
    layer itself into the type it computes in (``layer.to(torch.bfloat16)``), or cast its input."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", device=None,
                 dtype=None):
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear(input, self.weight, self.bias, self.activation, residual)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
