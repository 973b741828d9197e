"""Refusals of the linear layer, the gradient norm and clipping: wrong arguments end in an error before anything is
launched, in Python and at the C interface.  Nothing here needs a GPU."""
import contextlib
import ctypes

import numpy as np
import pytest
import torch

import vq_vae_amd as vq
from vq_vae_amd import _lib, projection

BF, F32 = torch.bfloat16, torch.float32


def t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args, kwargs, error, says", [
    ((t(2, 3), t(4, 3)), {}, RuntimeError, "GPU"),
    ((t(2, 3), t(4, 3)), {"activation": "tanh"}, ValueError, "activation"),
    ((t(2, 3), t(4, 5)), {}, ValueError, "in features"),
    ((t(2, 3), t(3)), {}, ValueError, "weight"),
    ((t(2, 3), t(0, 3)), {}, ValueError, "weight"),
    ((t(2, 0), t(4, 0)), {}, ValueError, "weight"),
    ((t(2, 3), t(4, 3, dtype=BF)), {}, TypeError, "share one type"),
    ((t(2, 3), t(4, 3), t(4, dtype=BF)), {}, TypeError, "share one type"),
    ((t(2, 3, dtype=torch.float64), t(4, 3, dtype=torch.float64)), {}, TypeError, "float64"),
    ((t(2, 3), t(4, 3), t(3)), {}, ValueError, "bias"),
    ((t(2, 3), t(4, 3), t(1, 4)), {}, ValueError, "bias"),
    ((t(2, 3), t(4, 3)), {"residual": t(2, 3)}, ValueError, "residual"),
    ((t(2, 3), t(4, 3)), {"residual": t(1, 4)}, ValueError, "residual"),        # nothing is broadcast
    ((t(2, 3), t(4, 3)), {"residual": t(4)}, ValueError, "residual"),
    ((t(()), t(4, 3)), {}, ValueError, "in features"),
    ((np.zeros((2, 3)), t(4, 3)), {}, TypeError, "tensor"),
    ((t(2, 3), None), {}, TypeError, "weight"),
    ((torch.zeros(1, 1).expand(1, (1 << 20) + 1), torch.zeros(1, 1).expand(1, (1 << 20) + 1)), {}, ValueError, "up to"),
])
def test_linear_refuses(args, kwargs, error, says):
    with pytest.raises(error, match=says):
        vq.linear(*args, **kwargs)


def test_layer_has_the_parameters_of_a_linear_layer():
    a, b = vq.Linear(5, 7, activation="silu"), torch.nn.Linear(5, 7)
    assert {k: v.shape for k, v in a.state_dict().items()} == {k: v.shape for k, v in b.state_dict().items()}
    a.load_state_dict(b.state_dict())
    assert "silu" in repr(a)
    with pytest.raises(ValueError, match="activation"):
        vq.Linear(5, 7, activation="sine")


def test_gradient_functions_refuse():
    g = [t(3), t(4)]
    with pytest.raises(RuntimeError, match="GPU"):
        vq.grad_norm(g)
    with pytest.raises(RuntimeError, match="GPU"):
        vq.clip_grads(g, 1.0)
    for bad in (0, 3, -1.0, float("nan")):
        with pytest.raises(ValueError, match="norm_type"):
            vq.grad_norm(g, bad)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            vq.clip_grads(g, bad)
    with pytest.raises(TypeError, match="float64"):
        vq.grad_norm([t(3, dtype=torch.float64)])
    with pytest.raises(TypeError, match="tensors"):
        vq.grad_norm([t(3), None])
    with pytest.raises(TypeError, match="dense"):
        vq.grad_norm([t(3, 3).to_sparse()])
    with pytest.raises(ValueError, match="one device"):
        vq.grad_norm([t(3), torch.zeros(3, device="meta")])


def test_clipping_refuses_shared_and_expanded_memory():
    a = t(6, 4)
    for bad in ([a, a], [a, a[2:3]], [a[:, :2], a[:, 1:3]], [a, a.t()], [a.view(-1)[:5], a.view(-1)[4:]]):
        with pytest.raises(ValueError, match="share memory"):
            vq.clip_grads(bad, 1.0)
    with pytest.raises(ValueError, match="expanded"):
        vq.clip_grads([t(1, 4).expand(3, 4)], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        vq.clip_grads([a[0], a[1]], 1.0, out=[a[1], a[0]])
    with pytest.raises(ValueError, match="share memory"):       # 16-bit gradients in the first half of their own fp32 output
        vq.clip_grads([a.view(-1).view(BF)[:24]], 1.0, out=[a.view(-1)])
    # neighbours in one buffer are apart
    with pytest.raises(RuntimeError, match="GPU"):
        vq.clip_grads([a[:3], a[3:]], 1.0)


def test_clipping_refuses_wrong_outputs():
    with pytest.raises(ValueError, match="1 gradients but 2"):
        vq.clip_grads([t(3)], 1.0, out=[t(3), t(3)])
    with pytest.raises(ValueError, match="shape"):
        vq.clip_grads([t(3)], 1.0, out=[t(4)])
    with pytest.raises(TypeError, match="same type or float32"):
        vq.clip_grads([t(3)], 1.0, out=[t(3, dtype=BF)])
    with pytest.raises(ValueError, match="requires a gradient"):
        vq.clip_grads([t(3)], 1.0, out=[t(3).requires_grad_()])


def test_nothing_to_clip():
    assert float(vq.grad_norm([])) == 0.0
    assert float(vq.clip_grads([], 1.0)) == 0.0
    p = torch.nn.Parameter(t(3))
    assert float(vq.clip_grad_norm_([p], 1.0)) == 0.0
    with pytest.raises(ValueError, match="max_norm"):
        vq.clip_grad_norm_([p], -1.0)


INVALID, UNSUPPORTED, TOO_LARGE = 1, 2, 3


def test_c_interface_checks_its_arguments():
    lib = _lib.load()
    p = ctypes.c_void_p(4096)                  # never followed: every call below ends at its checks
    ok = (p, 8, p, 8, None, None, 0, 0, 0, 4, 8, 8, p, None, p, None)

    def linear(**kw):
        names = "x ldx W ldw bias residual ldr dtype act M K N y pre work stream".split()
        return lib.vq_linear(*(kw.get(n, v) for n, v in zip(names, ok)))

    for kw in ({"x": None}, {"W": None}, {"y": None}, {"M": -1}, {"K": 0}, {"N": 0}, {"dtype": 3}, {"dtype": -1}, {"act": 5},
               {"act": -1}, {"ldx": 7}, {"ldw": 7}, {"residual": p, "ldr": 7}):
        assert linear(**kw) == INVALID, kw
    assert linear(K=(1 << 20) + 1, ldx=1 << 21, ldw=1 << 21) == UNSUPPORTED
    assert linear(ldx=1 << 22) == UNSUPPORTED
    assert linear(M=(1 << 31) + 1) == UNSUPPORTED
    assert linear(M=0, x=None, y=None) == 0
    assert lib.vq_linear_act_grad(p, p, 0, 0, 8, p, None) == INVALID      # no activation has no gradient to apply
    assert lib.vq_linear_act_grad(None, p, 0, 1, 8, p, None) == INVALID
    assert lib.vq_linear_act_grad(p, p, 0, 1, -1, p, None) == INVALID
    assert lib.vq_linear_act_grad(None, None, 0, 1, 0, None, None) == 0
    assert lib.vq_linear_dgrad(None, p, 8, 0, 4, 8, 8, p, p, None) == INVALID
    assert lib.vq_linear_dgrad(p, p, 7, 0, 4, 8, 8, p, p, None) == INVALID
    assert lib.vq_linear_dgrad(None, p, 8, 0, 0, 8, 8, None, p, None) == 0
    assert lib.vq_linear_wgrad(p, p, 8, 0, 4, 8, 8, None, None, p, None) == INVALID
    assert lib.vq_linear_wgrad(p, None, 8, 0, 4, 8, 8, p, None, p, None) == INVALID
    assert lib.vq_linear_wgrad(p, p, 8, 0, 4, 8, 8, None, p, None, None) == INVALID     # the column sums need work
    back = (p, p, p, 8, p, 8, 0, 1, 4, 8, 8, p, p, p, p, None)
    for at, v in ((0, None), (1, None), (3, 7), (5, 7), (6, 3), (7, 5), (8, -1), (9, 0), (10, 0), (14, None), (14, ctypes.c_void_p(4104))):
        assert lib.vq_linear_backward(*(v if i == at else a for i, a in enumerate(back))) in (INVALID, ), (at, v)
    # a split sum without its workspace
    assert lib.vq_linear_work_bytes(2, 1 << 20, 64, 64, 1) > 0
    assert lib.vq_linear_wgrad(p, p, 64, 1, 1 << 20, 64, 64, p, None, None, None) == INVALID
    for bad in ((4, 4, 8, 8, 0), (-1, 4, 8, 8, 0), (0, -1, 8, 8, 0), (0, 4, 0, 8, 0), (0, 4, 8, 8, 7)):
        assert lib.vq_linear_work_bytes(*bad) == 0


class Ref(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("numel", ctypes.c_int64), ("src_type", ctypes.c_int32),
                ("dst_type", ctypes.c_int32)]


def test_c_interface_checks_the_tensor_list():
    lib = _lib.load()
    p = ctypes.c_void_p(4096)

    def both(*refs, kind=2, max_norm=1.0, norm=p, work=p, n=None):
        arr = (Ref * max(1, len(refs)))(*refs)
        n = len(refs) if n is None else n
        return (lib.vq_grad_norm(arr, n, kind, norm, work, None), lib.vq_clip_grads(arr, n, kind, max_norm, norm, work, None))

    good = Ref(4096, 8192, 8, 0, 0)
    assert both(good, kind=3) == (INVALID, INVALID)
    assert both(good, kind=-1) == (INVALID, INVALID)
    assert both(good, norm=None) == (INVALID, INVALID)
    assert both(good, work=None) == (INVALID, INVALID)
    assert both(good, work=ctypes.c_void_p(4100)) == (INVALID, INVALID)
    assert both(good, n=-1) == (INVALID, INVALID)
    assert both(Ref(None, 8192, 8, 0, 0)) == (INVALID, INVALID)
    assert both(Ref(4096, 8192, -1, 0, 0)) == (INVALID, INVALID)
    assert both(Ref(4096, 8192, 8, 3, 3)) == (INVALID, INVALID)
    arr = (Ref * 1)(Ref(4096, None, 8, 0, 0))
    assert lib.vq_clip_grads(arr, 1, 2, 1.0, p, p, None) == INVALID
    arr = (Ref * 1)(Ref(4096, 8192, 8, 0, 1))          # fp32 into bf16
    assert lib.vq_clip_grads(arr, 1, 2, 1.0, p, p, None) == INVALID
    arr = (Ref * 1)(good)
    assert lib.vq_clip_grads(arr, 1, 2, -1.0, p, p, None) == INVALID
    assert lib.vq_clip_grads(arr, 1, 2, float("nan"), p, p, None) == INVALID
    many = (Ref * 65537)()
    assert lib.vq_grad_norm(many, 65537, 2, p, p, None) == TOO_LARGE
    assert lib.vq_grad_norm_work_bytes(-1) == 0 and lib.vq_grad_norm_work_bytes(0) > 0


class Products:
    """The calls of the library that a layer without activation makes, on host memory (fp32)."""

    @staticmethod
    def at(address, rows, cols, pitch):
        flat = np.ctypeslib.as_array((ctypes.c_float * ((rows - 1) * pitch + cols)).from_address(address))
        return np.lib.stride_tricks.as_strided(flat, (rows, cols), (4 * pitch, 4))

    def vq_linear(self, x, ldx, W, ldw, bias, residual, ldr, dtype, act, M, K, N, y, pre, work, stream):
        assert all(type(v) is int for v in (ldx, ldw, ldr, M, K, N))
        out = self.at(x, M, K, ldx) @ self.at(W, N, K, ldw).T
        if bias:
            out = out + self.at(bias, 1, N, N)
        if residual:
            out = out + self.at(residual, M, N, ldr)
        self.at(y, M, N, N)[:] = out
        return 0

    def vq_linear_backward(self, gy, pre, x, ldx, W, ldw, dtype, act, M, K, N, gx, gW, gbias, work, stream):
        g = self.at(gy, M, N, N)
        for to, shape, value in ((gx, (M, K), g @ self.at(W, N, K, ldw)), (gW, (N, K), g.T @ self.at(x, M, K, ldx)), (gbias, (1, N), g.sum(0))):
            if to:
                self.at(to, *shape, shape[1])[:] = value
        return 0


@pytest.fixture
def products(monkeypatch):
    """What the layer hands to the library, and what torch makes of it, without a GPU."""
    monkeypatch.setattr(projection._lib, "load", Products)
    monkeypatch.setattr(projection, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(projection, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(projection, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(projection, "_work_bytes", lambda *a: 0)


def layer_inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g) for s in ((7, 3), (4, 3), (4,), (7, 4))]


def formula(x, w, b, r):
    return x @ w.t() + b + r


def test_stand_in_for_the_library(products):
    args = [a.requires_grad_() for a in layer_inputs()]
    y, want = vq.linear(*args[:3], residual=args[3]), formula(*args)
    assert torch.allclose(y, want)
    for a, b in zip(torch.autograd.grad(y.square().sum(), args), torch.autograd.grad(want.square().sum(), args)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_derivatives_are_refused(products, requires_grad):
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        for i in range(4):
            args = [a.requires_grad_(requires_grad) for a in layer_inputs()]
            args[i] = fwad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                vq.linear(*args[:3], residual=args[3])
        # what carries no tangent is answered
        args = [a.requires_grad_(requires_grad) for a in layer_inputs()]
        y = vq.linear(*args[:3], residual=args[3])
        assert torch.allclose(y, formula(*args))
        # a tangent that arrives with the output's gradient
        if requires_grad:
            for at in (0, 3):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.autograd.grad(y, args[at], fwad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
        g = fwad.make_dual(torch.ones(3), torch.ones(3))
        for call in (lambda: vq.grad_norm([torch.ones(2), g]), lambda: vq.clip_grads([g], 1.0),
                     lambda: vq.clip_grads([torch.ones(3)], 1.0, out=[g])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.parametrize("requires_grad", [False, True])
def test_traces_are_refused(products, requires_grad):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    args = [a.requires_grad_(requires_grad) for a in layer_inputs()]
    for call in (lambda g: vq.linear(g, args[1]), lambda g: vq.grad_norm([g.detach()]), lambda g: vq.clip_grads([g.detach()], 1.0)):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call)(args[0])
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(call, args[0], check_trace=False)

    class Passing(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Passing():
        assert torch.allclose(vq.linear(*args[:3], residual=args[3]), formula(*args))


def test_the_norm_is_not_part_of_a_graph():
    # a penalty on it would contribute nothing: refused, not detached
    x = torch.ones(3, requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    for bad in ([g], [t(3), x]):
        with pytest.raises(RuntimeError, match="not differentiable"):
            vq.grad_norm(bad)
        for fine in (torch.no_grad(), torch.inference_mode()):
            with fine, pytest.raises(RuntimeError, match="GPU"):
                vq.grad_norm(bad)
        with pytest.raises(RuntimeError, match="GPU"):
            vq.grad_norm([b.detach() for b in bad])
    # torch's clipping takes such gradients, and so does this
    x.grad = g
    for error_if_nonfinite in (False, True):
        with pytest.raises(RuntimeError, match="GPU"):
            vq.clip_grad_norm_([x], 1.0, error_if_nonfinite=error_if_nonfinite)


def test_clipping_takes_views_that_share_no_element():
    a, c = t(6, 4), t(3, 8, 10)
    fine = ([a[:, :2], a[:, 2:]], [a[:, 0], a[:, 1:3], a[:, 3]], [a[::2], a[1::2]], [a.view(-1)[::3], a.view(-1)[1::3], a.view(-1)[2::3]],
            [c[:, :4, :5], c[:, 4:, :5], c[..., 5:]], [c[:, ::2, ::2], c[:, ::2, 1::2], c[:, 1::2]], [a.t()[:2], a.t()[2:]],
            [a[:2, :2], a[2:], a[:2, 2:]], [t(4096, 30)[:, k::7] for k in range(7)])
    for grads in fine:
        with pytest.raises(RuntimeError, match="GPU"):
            vq.clip_grads(grads, 1.0)
        with pytest.raises(RuntimeError, match="GPU"):      # in place by another view of the same memory
            vq.clip_grads(grads, 1.0, out=[g[...] for g in grads])
    with pytest.raises(RuntimeError, match="GPU"):
        vq.clip_grads([a[:, :2]], 1.0, out=[a[:, 2:]])
    for bad in ([a[:, :2], a[:, 1:]], [a[::2], a[2:4, :1]], [c[:, :4, :5], c[2, 3:, 4:]], [a.view(-1)[::3], a.view(-1)[::2]]):
        with pytest.raises(ValueError, match="share memory"):
            vq.clip_grads(bad, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        vq.clip_grads([a[:, :2]], 1.0, out=[a[:, 1:3]])
    with pytest.raises(ValueError, match="share memory"):
        vq.clip_grads([t(5, 8, dtype=BF)[:, :4]] + [a[:, :2]], 1.0, out=[a.view(-1)[:20].view(5, 4), a[:, 2:]])


def test_shared_elements_are_found_exactly():
    # against the bytes themselves, strided windows of one small buffer; a search that would take too long refuses
    from vq_vae_amd import gradients
    rng = np.random.default_rng(0)
    buf = torch.zeros(400, dtype=torch.int8)

    def window():
        while True:
            kind = (torch.float32, torch.bfloat16)[rng.integers(2)]
            shape, stride = rng.integers(1, 6, rng.integers(0, 4)), rng.integers(0, 14, 3)
            stride = stride[:len(shape)]
            end = int(((shape - 1) * stride).sum()) + 1
            room = buf.numel() // kind.itemsize - end
            if room >= 0:
                return torch.as_strided(buf.view(kind), tuple(map(int, shape)), tuple(map(int, stride)), int(rng.integers(0, room + 1)))

    def bytes_of(v):
        at = {0}
        for n, st in zip(v.shape, v.stride()):
            at = {p + k * st * v.element_size() for p in at for k in range(n)}
        return {v.data_ptr() + p + k for p in at for k in range(v.element_size())}
    seen = [0, 0]
    for _ in range(3000):
        a, b = window(), window()
        want = bool(bytes_of(a) & bytes_of(b))
        assert gradients._meet(gradients._runs(a), gradients._runs(b)) == want
        assert gradients._shared([a, b]) == want
        seen[want] += 1
    assert min(seen) > 500
    big = torch.zeros(1, dtype=torch.float32)
    far = lambda first, dims: (first, first + 4 + sum(d * (n - 1) for d, n in dims), 4, dims)
    assert gradients._meet(far(0, [(1000003 * 8, 4000), (1000033 * 8, 4000)]), far(4, [(999983 * 8, 4000), (999979 * 8, 4000)]))


def test_layer_under_autocast(products):
    # the types stay: nothing is cast, and an input of another type than the parameters' is refused
    layer, x = vq.Linear(3, 4), torch.randn(7, 3)
    with torch.autocast("cpu", dtype=BF):
        assert torch.nn.Linear(3, 4)(x.to(BF)).dtype is BF
        with pytest.raises(TypeError, match="share one type"):
            layer(x.to(BF))
        y = layer(x)
    assert y.dtype is F32 and torch.equal(y, layer(x))
