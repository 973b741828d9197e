"""The linear layer (product with bias, activation and residual) and its gradients against the formulas in 64 bits.

Tolerances are error bounds, element by element, u = 2^-24 being half a step of the fp32 sums and h half a step of the
tensors' type (fp32 2^-24, bf16 2^-8, fp16 2^-11, relative to the value; fp16 also 2^-25 near zero):
  * a sum of n products in fp32, in any order: (n + 1) u sum|a b|; the bias adds one rounding of the result;
  * the activation: at most 1.13 times the error of its argument (the largest slope, that of gelu), plus its own evaluation,
    at most 32 u (|p| + 1): a dozen operations, a 1-ulp exponential and reciprocal;
  * an output: h |y| + u (|p| + |r| ...) for its additions;
  * gradients: dp = gy act'(pre) has the error |gy| (0.8 (h |p| + error of p) + 32 u (|p| + 1)) -- 0.8 bounds |act''| -- and its
    own rounding h |dp|; for relu the slope may also be the other one where |p| is within its error of 0.  The two
    products carry that error through |W| and |x| and add their own.
"""
import math

import pytest
import torch

import vq_vae_amd as vq
from vq_vae_amd import _lib, ops

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def act64(p, act):
    if act == "none":
        return p, torch.ones_like(p)
    if act == "relu":
        return p.clamp(min=0), (p > 0).double()
    if act == "silu":
        s = torch.sigmoid(p)
        return p * s, s * (1 + p * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.special.erfc(-p / math.sqrt(2))
        return p * c, c + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (p + 0.044715 * p ** 3))
    return 0.5 * p * (1 + t), 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * k * (1 + 3 * 0.044715 * p * p)


def forward64(x, w, b, act, r):
    """y, pre, slope and the bounds of y and pre."""
    kind, K = x.dtype, x.shape[-1]
    h = HALF[kind]
    x, w = x.double(), w.double()
    p = x @ w.t()
    ep = (K + 1) * U * (x.abs() @ w.abs().t())
    if b is not None:
        p = p + b.double()
        ep = ep + U * p.abs()
    a, slope = act64(p, act)
    ey = 1.13 * ep + (32 * U * (p.abs() + 1) if act not in ("none", "relu") else 0)
    y = a
    if r is not None:
        y = y + r.double()
        ey = ey + U * y.abs()
    return y, p, slope, ey * 1.001 + h * y.abs() + TINY[kind], ep


def backward64(gy, x, w, p, ep, slope, act):
    """gradients of input, weight and bias with their bounds."""
    kind = x.dtype
    h, (M, K), N = HALF[kind], x.shape, w.shape[0]
    gy, x, w = gy.double(), x.double(), w.double()
    dp = gy * slope
    if act == "none":
        ed = torch.zeros_like(dp)
    else:
        d_slope = 0.8 * (h * p.abs() + TINY[kind] + ep) + 32 * U * (p.abs() + 1)
        if act == "relu":
            d_slope = (p.abs() <= ep + TINY[kind]).double()
        ed = gy.abs() * d_slope * 1.01 + h * dp.abs() * 1.01 + TINY[kind]
    gx, gw, gb = dp @ w, dp.t() @ x, dp.sum(0)
    ad = dp.abs() + ed
    ex = ed @ w.abs() + (N + 1) * U * (ad @ w.abs()) + h * 1.01 * gx.abs() + TINY[kind]
    ew = ed.t() @ x.abs() + (M + 1) * U * (ad.t() @ x.abs()) + h * 1.01 * gw.abs() + TINY[kind]
    eb = ed.sum(0) + (M + 1) * U * ad.sum(0) + h * 1.01 * gb.abs() + TINY[kind]
    return (gx, ex), (gw, ew), (gb, eb)


def close(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / bound).max()):.3g} of the bound "
                                 f"at {[int(v) for v in bad.nonzero()[0]]}")


def make(M, K, N, kind, bias, residual, strided, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(kind)
    x = normal(M, 2 * K)[:, K:] if strided else normal(M, K)
    w = normal(N, K + 5, scale=K ** -0.5)[:, :K] if strided else normal(N, K, scale=K ** -0.5)
    return x, w, normal(N) if bias else None, (normal(M, N + 3)[:, :N] if strided else normal(M, N)) if residual else None, normal(M, N)


# one row, a few, tiles that end inside, one element over a tile, reductions shorter than a step and split ones
SIZES = [(1, 1, 1), (1, 256, 1024), (2, 7, 5), (3, 64, 2), (16, 130, 33), (17, 64, 64), (5, 20000, 40), (40, 8192, 72), (63, 65, 66),
         (64, 64, 64), (129, 257, 127), (300, 515, 130), (1000, 96, 520), (777, 130, 515), (256, 512, 256), (2048, 40, 16),
         (515, 1024, 2048), (2049, 1032, 2056)]


@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(size, kind):
    M, K, N = size
    i = SIZES.index(size) + TYPES.index(kind)
    for act, bias, residual, strided in ((ACTS[i % 5], True, True, i % 2 == 1), (ACTS[(i + 2) % 5], i % 2 == 0, False, i % 2 == 0)):
        x, w, b, r, gy = make(M, K, N, kind, bias, residual, strided, 100 * i)
        y, p, slope, ey, ep = forward64(x, w, b, act, r)
        close(vq.linear(x, w, b, act, r), y, ey, "forward")
        leaves = [t.requires_grad_() for t in (x.detach(), w.detach(), b, r) if t is not None]
        x2, w2 = leaves[0], leaves[1]
        out = vq.linear(x2, w2, b, act, r)
        close(out.detach(), y, ey, "forward with gradients")
        grads = torch.autograd.grad(out, leaves, gy)
        (gx, ex), (gw, ew), (gb, eb) = backward64(gy, x, w, p, ep, slope, act)
        close(grads[0], gx, ex, "input gradient")
        close(grads[1], gw, ew, "weight gradient")
        if b is not None:
            close(grads[2], gb, eb, "bias gradient")
        if r is not None:
            assert torch.equal(grads[-1], gy)


@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
def test_every_activation(act, kind):
    # values from the tails to the middle: the product is one-hot, so that p is an input
    p = torch.cat([torch.linspace(-12, 12, 481), torch.tensor([0.0, -0.0, 1e-7, -1e-7, 60.0, -60.0, 200.0, -200.0])]).to(DEV, kind)
    x = p.view(-1, 1)
    w = torch.ones(1, 1, device=DEV, dtype=kind)
    y, q, slope, ey, ep = forward64(x, w, None, act, None)
    xr = x.clone().requires_grad_()
    out = vq.linear(xr, w, activation=act)
    close(out.detach(), y, ey, "forward")
    (gx,) = torch.autograd.grad(out, xr, torch.ones_like(out))
    (want, ex), _, _ = backward64(torch.ones_like(out), x, w, q, ep, slope, act)
    close(gx, want, ex, "gradient")


def test_differences():
    # along a random direction, fp32: the loss is summed in 64 bits; the step's error is h^2 f''' / 6 with f''' of order 1 per
    # element, the kernel's rounding error of y (1e-6 an element) is divided by 2 h
    x, w, b, r, gy = make(40, 33, 21, torch.float32, True, True, False, 5)
    for act in ("silu", "gelu", "gelu_tanh"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        out = vq.linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
        grads = torch.autograd.grad(out, leaves, gy)
        g = torch.Generator(device=DEV).manual_seed(9)
        step = 2.0 ** -7
        for t, gt in zip(leaves, grads):
            d = torch.randn(t.shape, generator=g, device=DEV)
            d /= d.abs().max()

            def loss(sign):
                args = [(u + sign * step * d if u is t else u).detach() for u in leaves]
                return (vq.linear(args[0], args[1], args[2], act, args[3]).double() * gy.double()).sum()
            num = float((loss(1) - loss(-1)) / (2 * step))
            ana = float((gt.double() * d.double()).sum())
            n = gy.abs().double().sum().item()
            # direction of x: |p'| <= sum|w| of about 4.6, of w: sum|x| of about 27; f''' <= 2 |p'|^3; errors of random sign add
            # like their square root
            reach = 4.6 if t is leaves[0] else 27.0 if t is leaves[1] else 1.0
            tol = math.sqrt(gy.numel()) * (step ** 2 / 6 * 2 * reach ** 3 + 4e-6 / step) + 1e-6 * n
            assert abs(num - ana) <= tol, (act, tuple(t.shape), num, ana, tol)


def test_shapes_without_rows_and_with_many_dimensions():
    w = torch.randn(5, 3, device=DEV, requires_grad=True)
    b = torch.randn(5, device=DEV, requires_grad=True)
    x = torch.zeros(0, 3, device=DEV, requires_grad=True)
    y = vq.linear(x, w, b, "silu")
    assert y.shape == (0, 5)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 5, device=DEV))
    assert gx.shape == (0, 3) and not gw.any() and not gb.any()
    (gb,) = torch.autograd.grad(vq.linear(x.detach(), w.detach(), b), b, torch.zeros(0, 5, device=DEV))
    assert not gb.any()
    v = torch.randn(2, 3, 4, 3, device=DEV)
    assert vq.linear(v, w, b).shape == (2, 3, 4, 5)
    assert torch.equal(vq.linear(v, w, b).view(24, 5), vq.linear(v.view(24, 3), w, b))
    assert vq.linear(v[0, 0, 0], w, b).shape == (5,)
    # other strides: transposed, expanded rows, transposed weight
    vt = v.transpose(1, 2)
    assert torch.equal(vq.linear(vt, w, b), vq.linear(vt.contiguous(), w, b))
    e = torch.randn(1, 3, device=DEV).expand(70, 3)
    assert torch.equal(vq.linear(e, w, b), vq.linear(e.contiguous(), w, b))
    wt = torch.randn(3, 5, device=DEV).t()
    assert torch.equal(vq.linear(v, wt, b), vq.linear(v, wt.contiguous(), b))


def test_expanded_inputs_have_summed_gradients():
    # autograd reduces what expand broadcast; grad_output itself may be expanded too (a sum's gradient)
    w = torch.randn(66, 40, device=DEV, requires_grad=True)
    row = torch.randn(40, device=DEV, requires_grad=True)
    res = torch.randn(66, device=DEV, requires_grad=True)
    y = vq.linear(row.expand(100, 40), w, activation="gelu", residual=res.expand(100, 66))
    g = torch.autograd.grad(y.sum(), (row, w, res))
    rd, wd = row.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = torch.autograd.grad(torch.nn.functional.gelu(rd.expand(100, 40) @ wd.t()).sum(), (rd, wd))
    for a, b in zip(g, want):      # 100 equal terms, each within 1e-5 of the scale of the gradient
        assert float((a.double() - b).abs().max()) <= 2e-5 * float(b.abs().max())
    assert torch.equal(g[2], torch.full_like(g[2], 100.0))


@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M", [5, 100])
def test_nonfinite_rows_stay_among_themselves(M, kind):
    K, N = 70, 66
    x, w, b, r, gy = make(M, K, N, kind, True, True, False, 3)
    clean = vq.linear(x, w, b, "silu", r)
    x[2, 5] = float("nan")
    x[4, 69] = float("inf")
    y = vq.linear(x, w, b, "silu", r)
    keep = [i for i in range(M) if i not in (2, 4)]
    assert torch.equal(y[keep], clean[keep])
    assert bool(y[2].isnan().all()) and not bool(y[4].isfinite().all())
    # a weight row: one output column
    x, w, b, r, gy = make(M, K, N, kind, True, True, False, 3)
    w[7, 0] = float("nan")
    y = vq.linear(x, w, b, "silu", r)
    cols = [j for j in range(N) if j != 7]
    assert torch.equal(y[:, cols], clean[:, cols]) and bool(y[:, 7].isnan().all())
    # relu keeps a NaN, as max(p, 0) with a NaN does
    assert bool(vq.linear(x, w, b, "relu")[:, 7].isnan().all())


def test_half_precision_beyond_its_range():
    # pre is kept in fp16: beyond its range it is infinite, and the slope there is its limit, not inf * 0
    x = torch.full((20, 64), 200.0, device=DEV, dtype=torch.float16, requires_grad=True)
    w = torch.full((8, 64), 100.0, device=DEV, dtype=torch.float16, requires_grad=True)
    for act in ACTS[1:]:
        y = vq.linear(x, w, activation=act)
        (gx,) = torch.autograd.grad(y, x, torch.full_like(y, 2.0 ** -6))
        assert bool((gx == 100.0 * 8 * 2.0 ** -6).all()), act
        y = vq.linear(x, -w.detach(), activation=act)
        (gx,) = torch.autograd.grad(y, x, torch.full_like(y, 2.0 ** -6))
        assert bool((gx == 0).all()), act


def test_nothing_outside_the_outputs_is_written():
    # through the C interface, outputs in the middle of larger buffers
    lib = _lib.load()
    for M, K, N, dt, kind in ((3, 40, 50, 1, torch.bfloat16), (65, 72, 129, 1, torch.bfloat16), (130, 33, 70, 0, torch.float32),
                              (300, 256, 520, 2, torch.float16), (40, 4096, 65, 1, torch.bfloat16)):
        x, w, b, r, gy = make(M, K, N, kind, True, True, False, 1)
        s = ops._stream(DEV)

        def band(n):
            buf = torch.full((n + 128,), 7.0, device=DEV, dtype=kind)
            return buf, buf[64:64 + n]
        (yb, y), (pb, p), (xb, gx), (wb, gw), (bb, gb) = (band(n) for n in (M * N, M * N, M * K, N * K, N))
        work = [torch.empty(max(16, lib.vq_linear_work_bytes(q, M, K, N, dt)), dtype=torch.uint8, device=DEV) for q in range(3)]
        P = ops._ptr
        assert lib.vq_linear(P(x), K, P(w), K, P(b), P(r), N, dt, 2, M, K, N, P(y), P(p), P(work[0]), s) == 0
        assert lib.vq_linear_dgrad(P(gy), P(w), K, dt, M, K, N, P(gx), P(work[1]), s) == 0
        assert lib.vq_linear_wgrad(P(gy), P(x), K, dt, M, K, N, P(gw), P(gb), P(work[2]), s) == 0
        torch.cuda.synchronize()
        for buf in (yb, pb, xb, wb, bb):
            assert bool((buf[:64] == 7).all()) and bool((buf[-64:] == 7).all())
        assert torch.equal(y.view(M, N), vq.linear(x, w, b, "silu", r))
        # the bias gradient alone comes from another kernel: the same sums up to their order
        gb2 = torch.empty(N, device=DEV, dtype=kind)
        assert lib.vq_linear_wgrad(P(gy), None, K, dt, M, K, N, None, P(gb2), P(work[2]), s) == 0
        ref = gy.double().sum(0)
        bound = (M + 1) * U * gy.double().abs().sum(0) + 1.01 * HALF[kind] * ref.abs() + TINY[kind]
        close(gb, ref, bound, "bias gradient")
        close(gb2, ref, bound, "bias gradient alone")


def test_partial_gradients():
    x, w, b, r, gy = make(200, 64, 96, torch.bfloat16, True, True, False, 8)
    full = {}
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    out = vq.linear(x, w, b, "gelu", r)
    for t, g in zip(leaves, torch.autograd.grad(out, leaves, gy)):
        full[id(t)] = g
    for chosen in ([0], [1], [0, 1], [0, 2], [3], [1, 3]):
        for i, t in enumerate(leaves):
            t.requires_grad_(i in chosen)
        out = vq.linear(x, w, b, "gelu", r)
        for i, g in zip(chosen, torch.autograd.grad(out, [leaves[i] for i in chosen], gy)):
            assert torch.equal(g, full[id(leaves[i])])
    for t in leaves:
        t.requires_grad_(False)
    b.requires_grad_()
    (gb,) = torch.autograd.grad(vq.linear(x, w, b, "gelu", r), [b], gy)
    # the sums of the same 200 rounded terms in another order, rounded to bf16
    assert float((gb.float() - full[id(b)].float()).abs().max()) <= 2.0 ** -7 * float(full[id(b)].float().abs().max())
    with pytest.raises(RuntimeError):      # differentiable once
        x.requires_grad_()
        (gx,) = torch.autograd.grad(vq.linear(x, w, b, "gelu").float().sum(), [x], create_graph=True)
        torch.autograd.grad(gx.float().sum(), [x])


def test_same_bits_on_every_run():
    x, w, b, r, gy = make(3000, 520, 264, torch.bfloat16, True, True, False, 4)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    runs = []
    for _ in range(3):
        out = vq.linear(x, w, b, "silu", r)
        runs.append([out.detach(), *torch.autograd.grad(out, leaves, gy)])
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))


def test_large_offsets():
    # inputs and outputs of more than 2^31 elements (4 GiB and more): rows at the start, in the middle and at the end
    M, K, N = 2 ** 21 + 3, 1032, 1040
    w = torch.randn(N, K, device=DEV).mul_(K ** -0.5).bfloat16()
    b = torch.randn(N, device=DEV).bfloat16()
    x = torch.empty(M, K, device=DEV, dtype=torch.bfloat16)
    for part in x.split(2 ** 18):
        part.copy_(torch.randn(part.shape, device=DEV))
    y = vq.linear(x, w, b, "silu")
    rows = torch.tensor([0, 1, 2 ** 20 - 1, 2 ** 20, M // 2, 2 ** 21 - 1, 2 ** 21, M - 2, M - 1], device=DEV)
    want, _, _, ey, _ = forward64(x[rows], w, b, "silu", None)
    close(y[rows], want, ey, "forward")
    # weight gradient: a sum over all rows.  gy is one at chosen rows, zero elsewhere
    gy = y.zero_()
    gy[rows] = 1.0
    w.requires_grad_()
    xg = x.requires_grad_()
    gx, gw = torch.autograd.grad(vq.linear(xg, w), [xg, w], gy)
    want = x.detach()[rows].double().sum(0).expand(N, K)
    bound = 10 * U * x.detach()[rows].double().abs().sum(0).expand(N, K) + HALF[torch.bfloat16] * 1.01 * want.abs() + 1e-30
    close(gw, want, bound, "weight gradient")
    wsum = w.detach().double().sum(0)
    bound = (N + 1) * U * w.detach().double().abs().sum(0) + HALF[torch.bfloat16] * 1.01 * wsum.abs() + 1e-30
    close(gx[rows], wsum.expand(len(rows), K), bound.expand(len(rows), K), "input gradient")
    assert not bool(gx[rows[-1] - 2 - 5].any())


def test_other_stream_and_layer():
    layer = vq.Linear(72, 40, activation="gelu").to(DEV, torch.bfloat16)
    x = torch.randn(33, 72, device=DEV).bfloat16()
    r = torch.randn(33, 40, device=DEV).bfloat16()
    want = layer(x, r)
    assert torch.equal(want, vq.linear(x, layer.weight, layer.bias, "gelu", r))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [layer(x, r) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want, o) for o in outs)
    with torch.autocast("cuda", dtype=torch.float16):       # the tensors' types stay
        assert torch.equal(layer(x, r), want)


@pytest.mark.parametrize("M", [4, 700])
def test_captured_and_replayed(M):
    # forward and backward in two graphs with memory of their own, replayed in turn between eager work, on new inputs
    kind, K, N = torch.bfloat16, 264, 136
    w = torch.randn(N, K, device=DEV).mul_(0.06).to(kind).requires_grad_()
    b = torch.randn(N, device=DEV).to(kind).requires_grad_()

    def step(x, r, gy):
        y = vq.linear(x, w, b, "gelu", r)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), gy))

    def inputs(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        return [torch.randn(*s, generator=g, device=DEV).to(kind) for s in ((M, K), (M, N), (M, N))]

    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = [[t.requires_grad_(i == 0) for i, t in enumerate(inputs(k))] for k in range(2)]
        step(*held[0])
    torch.cuda.current_stream().wait_stream(side)
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held[k])
        graphs.append((graph, held[k], out))
    for n in range(3):
        for k, (graph, ins, outs) in enumerate(graphs):
            new = inputs(10 * n + k + 5)
            with torch.no_grad():
                for t, v in zip(ins, new):
                    t.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            want = step(new[0].requires_grad_(), *new[1:])
            for o, e in zip(outs, want):
                assert torch.equal(o, e)


@pytest.mark.parametrize("act", ["none", "gelu"])
def test_hooks_on_saved_tensors(act):
    # a hook may bring a saved tensor back with other strides (copied away and back, as offloading does): the gradients are
    # those without it; one of another shape, type or device is refused
    M, K, N = 70, 40, 24
    x, w, b, r, gy = make(M, K, N, torch.bfloat16, True, True, True, 6)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def run(pack, unpack, gy=gy):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = vq.linear(x, w, b, act, r)
        return torch.autograd.grad(y, leaves, gy)
    want = run(lambda t: t, lambda t: t)
    turned = gy.t().contiguous().t()
    away = lambda t: t.cpu().contiguous()
    for got in (run(away, lambda t: t.to(DEV)), run(away, lambda t: t.to(DEV).t().contiguous().t()),
                run(lambda t: t, lambda t: t, turned), run(away, lambda t: t.to(DEV), turned)):
        assert all(torch.equal(a, c) for a, c in zip(want, got))
    for wrong in (lambda t: t, lambda t: t.to(DEV).float(), lambda t: t.to(DEV)[:, 1:], lambda t: t.to(DEV)[1:]):
        with pytest.raises(RuntimeError, match="hook on saved tensors"):
            run(away, wrong)


def test_recomputed_in_the_backward_pass():
    # checkpointing hands the backward pass tensors of a second forward pass
    from torch.utils.checkpoint import checkpoint
    x, w, b, r, gy = make(33, 40, 24, torch.float16, True, True, False, 9)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    f = lambda x, r: vq.linear(vq.linear(x, w, b, "silu", r), w.t()[:, :24], None, "gelu")   # the second weight is copied first
    def grads(out):
        return torch.autograd.grad(out, leaves, torch.ones_like(out))
    want = grads(f(x, r))
    assert all(torch.equal(a, c) for a, c in zip(want, grads(checkpoint(f, x, r, use_reentrant=False))))


def test_first_calls_of_a_process_captured():
    # a process of its own, where nothing of the library has run before the capture
    import subprocess
    import sys
    code = """
import torch, vq_vae_amd as vq
x = torch.randn(300, 264, device="cuda").half(); w = torch.randn(136, 264, device="cuda").half()
g = [torch.randn(5000, device="cuda"), torch.randn(70, device="cuda").half()]
big = [torch.randn(2048, 1024, device="cuda").bfloat16() for _ in range(2)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, z, n = vq.linear(x, w, None, "silu"), vq.linear(big[0], big[1]), vq.clip_grads(g, 1e9)
for _ in range(3):
    y.zero_(); z.zero_(); n.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, vq.linear(x, w, None, "silu")) and torch.equal(z, vq.linear(big[0], big[1])) and torch.equal(n, vq.grad_norm(g))
print("same")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]


@pytest.mark.parametrize("M, N", [(1, 1), (3, 7), (40, 33), (777, 515), (5000, 64), (4099, 1032), (100, 5000), (70, 9001)])
@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
def test_bias_gradient_is_summed_before_rounding(M, N, kind):
    # gy act'(pre) is rounded to the tensors' type for the products, but not for the bias gradient.  Against the formula at the
    # pre that the forward pass kept: 32 u (|p| + 1) for the slope, a rounding of the product, the fp32 sum, one rounding at the
    # end.  Alternating signs make the sum small beside its terms, where rounded terms would show.
    from vq_vae_amd import projection
    K = 16
    x, w, b, _, gy = make(M, K, N, kind, True, False, False, M + N)
    gy = gy.abs() * (1 - 2 * (torch.arange(M, device=DEV) % 2).to(kind))[:, None]
    for act in ("silu", "gelu"):
        _, pre = projection.linear_forward(x, w, b, act, want_pre=True)
        _, _, gb = projection.linear_backward(gy, x, w, pre, act, False, M % 2 == 1, True)
        p = pre.double()
        _, slope = act64(p, act)
        d = gy.double() * slope
        each = gy.double().abs() * 32 * U * (p.abs() + 1) + U * d.abs()
        bound = (each.sum(0) + (M + 1) * U * (d.abs() + each).sum(0)) * 1.001 + HALF[kind] * 1.01 * d.sum(0).abs() + TINY[kind]
        close(gb, d.sum(0), bound, f"{act}")


@pytest.mark.parametrize("M, K, N", [(1, 1, 1), (3, 40, 50), (70, 33, 2500), (777, 130, 515), (300, 256, 520), (40, 16, 9001)])
@pytest.mark.parametrize("kind, dt", [(torch.float32, 0), (torch.bfloat16, 1)], ids=["f32", "bf16"])
def test_backward_stays_within_its_outputs_and_workspace(M, K, N, kind, dt):
    lib = _lib.load()
    x, w, _, _, gy = make(M, K, N, kind, False, False, False, 2)
    pre = torch.nn.functional.linear(x.float(), w.float()).to(torch.float16 if kind is torch.bfloat16 else kind)   # as it is kept for silu
    bytes_of = lambda n: n * kind.itemsize

    def band(n):       # 256 bytes on either side
        buf = torch.full((n + 512,), 0x5a, device=DEV, dtype=torch.uint8)
        return buf, buf.data_ptr() + 256
    n_work = lib.vq_linear_work_bytes(3, M, K, N, dt)
    bands = [band(n) for n in (bytes_of(M * K), bytes_of(N * K), bytes_of(N), n_work)]
    P = ops._ptr
    assert lib.vq_linear_backward(P(gy), P(pre), P(x), K, P(w), K, dt, 2, M, K, N, *(p for _, p in bands), ops._stream(DEV)) == 0
    torch.cuda.synchronize()
    for buf, _ in bands:
        assert bool((buf[:256] == 0x5a).all()) and bool((buf[-256:] == 0x5a).all())
    p, (_, slope) = pre.double(), act64(pre.double(), "silu")
    (gx, ex), (gw, ew), (gb, eb) = backward64(gy, x, w, p, torch.zeros_like(p), slope, "silu")
    for (buf, _), want, bound, what in zip(bands, (gx, gw, gb), (ex, ew, eb), ("input", "weight", "bias")):
        close(buf[256:-256].view(kind).view(want.shape), want, bound, what)


@pytest.mark.parametrize("M", [4, 40])
def test_bf16_beyond_the_range_of_fp16(M):
    # p is kept in fp16 for a bf16 layer: infinite beyond 65504, where every slope has its limit; for relu the smallest p counts
    one = torch.ones(M, 64, device=DEV, dtype=torch.bfloat16)
    for size in (1e3, 1e6, 1e30):
        for act in ACTS[1:]:
            for sign in (1.0, -1.0):
                w = torch.full((8, 64), sign * size, device=DEV, dtype=torch.bfloat16)
                x = one.clone().requires_grad_()
                (gx,) = torch.autograd.grad(vq.linear(x, w, activation=act), x, torch.ones(M, 8, device=DEV, dtype=torch.bfloat16))
                want = 8.0 * float(w[0, 0]) if sign > 0 else 0.0
                assert bool((gx == want).all()), (size, act, sign)
    for tiny in (1e-9, 1e-30):
        for sign in (1.0, -1.0):
            w = torch.full((8, 64), sign * tiny, device=DEV, dtype=torch.bfloat16)
            x = one.clone().requires_grad_()
            (gx,) = torch.autograd.grad(vq.linear(x, w, activation="relu"), x, torch.ones(M, 8, device=DEV, dtype=torch.bfloat16))
            assert bool((gx == (8.0 * float(w[0, 0]) if sign > 0 else 0.0)).all())


def test_threads_on_streams_of_their_own():
    import threading
    sizes = [(300, 264, 136), (16, 8192, 512), (777, 130, 515), (2048, 256, 512)]
    cases = [make(*size, torch.bfloat16, True, True, False, 20 + i) for i, size in enumerate(sizes)]

    def step(case):
        x, w, b, r, gy = case
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = vq.linear(*leaves, "silu", r)
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]
    want = [step(c) for c in cases]
    norms = [vq.grad_norm(w[1:]) for w in want]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step(cases[i])
                    norm = vq.grad_norm(got[1:])
                    torch.cuda.current_stream().synchronize()
                    if not (all(torch.equal(a, c) for a, c in zip(got, want[i])) and torch.equal(norm, norms[i])):
                        wrong.append(i)
        except Exception as e:      # would be lost with the thread
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# few rows; tiles by DMA; by registers; a split sum joined; the 256 tile
@pytest.mark.parametrize("M, K, N", [(5, 70, 66), (100, 64, 72), (100, 70, 66), (40, 8192, 72), (2048, 64, 2048)])
@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
def test_activations_of_infinities_and_of_the_largest_values(M, K, N, kind):
    # p is one of the values exactly: one input channel with a weight of one, and the bias of a product of zeros
    top = torch.finfo(kind).max
    values = torch.tensor([math.inf, -math.inf, math.nan, top, -top], device=DEV).to(kind)
    by_row, by_col = values[torch.arange(M, device=DEV) % 5][:, None].expand(M, N), values[torch.arange(N, device=DEV) % 5].expand(M, N)
    x = torch.zeros(M, K, device=DEV, dtype=kind)
    w = torch.zeros(N, K, device=DEV, dtype=kind)
    w[:, 0] = 1.0
    hot = x.clone()
    hot[:, 0] = by_row[:, 0]
    for act in ACTS:
        for got, p in ((vq.linear(hot, w, None, act), by_row), (vq.linear(x, w, by_col[0].contiguous(), act), by_col)):
            want = act64(p.double(), act)[0]
            assert torch.equal(got.isnan(), want.isnan()), act
            assert torch.equal(got.isinf(), want.isinf()), act
            # largest values: act(p) is p or, below, less than the smallest number
            assert torch.equal(got.nan_to_num(nan=7.0).double(), want.to(kind).nan_to_num(nan=7.0).double()), act


@pytest.mark.parametrize("requires_grad", [False, True])
def test_recorded_calls(requires_grad):
    # a trace and a tangent are refused; a compiler runs the call outside its graphs
    import torch.autograd.forward_ad as fwad
    x, w, b, r, gy = make(40, 33, 21, torch.float32, True, True, False, 5)
    new = make(70, 33, 21, torch.float32, True, True, True, 6)
    f = lambda x, w, b, r: vq.linear(x, w, b, "gelu", r) * 2
    args = [t.clone().requires_grad_(requires_grad) for t in (x, w, b, r)]
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(f, args, check_trace=False)
    compiled = torch.compile(f, backend="eager")
    for tensors in ((x, w, b, r, gy), new):
        ins = [t.detach().clone().requires_grad_() for t in tensors[:4]]
        assert torch.equal(compiled(*tensors[:4]), f(*tensors[:4]))
        for a, c in zip(torch.autograd.grad(compiled(*ins), ins, tensors[4]), torch.autograd.grad(f(*ins), ins, tensors[4])):
            assert torch.equal(a, c)
    with fwad.dual_level():
        for i in range(4):
            dual = [fwad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError):
                f(*dual)
        with pytest.raises(NotImplementedError):
            vq.grad_norm([fwad.make_dual(x, x)])
        assert torch.equal(f(*args), f(x, w, b, r))


@pytest.mark.parametrize("M, K", [(4, 64), (40, 64), (40, 70), (40, 8192)])
@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
def test_relu_slope_of_the_smallest_values(M, K, kind):
    # p = +-2^-27 is nothing in fp16, but above or below zero: the slope is 1 or 0
    x = torch.zeros(M, K, device=DEV, dtype=kind)
    x[:, 0] = 2.0 ** -13
    x.requires_grad_()
    for sign in (1.0, -1.0, 0.0, -0.0):
        w = torch.zeros(72, K, device=DEV, dtype=kind)
        w[:, 0] = sign * 2.0 ** -14
        (gx,) = torch.autograd.grad(vq.linear(x, w, activation="relu"), x, torch.ones(M, 72, device=DEV, dtype=kind))
        assert bool((gx[:, 0] == (72 * 2.0 ** -14 if sign > 0 else 0.0)).all()) and not bool(gx[:, 1:].any()), sign


@pytest.mark.parametrize("kind, M", [(torch.float32, 2 ** 29 + 77), (torch.float16, 2 ** 29 + 77), (torch.bfloat16, 2 ** 31)],
                         ids=["f32", "f16", "bf16"])
def test_narrow_rows_to_two_to_the_31(kind, M):
    # more tiles of 64 rows than 2^23, to the most rows there may be.  Rows at both ends and round every power of two between
    K, N = 4, 3
    w = torch.randn(N, K, device=DEV).to(kind)
    b = torch.randn(N, device=DEV).to(kind)
    x = torch.empty(M, K, device=DEV, dtype=kind)
    for part in x.split(2 ** 26):
        part.copy_(torch.randn(2 ** 16, K, device=DEV).repeat(2 ** 10, 1)[:len(part)])
    rows = torch.tensor(sorted({0, 1, M - 1, M - 2, M - 78, *(2 ** k + d for k in range(20, 32) for d in (-1, 0, 1) if 2 ** k + d < M)}), device=DEV)
    y = vq.linear(x, w, b, "relu")
    want, _, _, ey, _ = forward64(x[rows], w, b, "relu", None)
    close(y[rows], want, ey, "forward")
    # every row, against the product of the 2^16 rows that a part repeats
    for i in (0, 3, M - 1 >> 26):
        part = x[i * 2 ** 26:(i + 1) * 2 ** 26]
        one = vq.linear(part[:2 ** 16], w, b, "relu")
        assert torch.equal(y[i * 2 ** 26:i * 2 ** 26 + len(part)], one.repeat(2 ** 10, 1)[:len(part)])
    del y
    # gradients: gy is one at those rows, zero elsewhere
    gy = torch.zeros(M, N, device=DEV, dtype=kind)
    gy[rows] = 1.0
    xg, wg = x.requires_grad_(), w.requires_grad_()
    gx, gw = torch.autograd.grad(vq.linear(xg, wg), [xg, wg], gy)
    want = x.detach()[rows].double().sum(0).expand(N, K)
    bound = 50 * U * x.detach()[rows].double().abs().sum(0).expand(N, K) + HALF[kind] * 1.01 * want.abs() + 1e-30
    close(gw, want, bound, "weight gradient")
    wsum = w.detach().double().sum(0)
    bound = (N + 1) * U * w.detach().double().abs().sum(0) + HALF[kind] * 1.01 * wsum.abs() + TINY[kind]
    close(gx[rows], wsum.expand(len(rows), K), bound.expand(len(rows), K), "input gradient")
    gx[rows] = 0
    assert not bool(gx.any())


@pytest.mark.parametrize("M", [16, 3000])
@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_tails_of_the_activations(act, kind, M):
    """Relative to the value, so that a tail which is lost shows.  With s = 1 / (1 + exp(-v)), q = |v| and a 1-ulp exponential
    and reciprocal (2 u each), v exact up to 4 u: 1 + exp and p s round twice, exp carries q times v's error and, as 2^(v log2 e), two
    roundings of its own argument: (8 + 7 q) u.  v = p for silu, p (a + b p^2) for gelu_tanh.
    Phi by erfc(z) = t exp(fit(t) - z^2), z = |p| / sqrt 2, t = 1 / (1 + z / 2): the fit 2 u; z 1.3 u, which moves erfc by 1 + 2 z^2 times
    that; t 3 u, and 1.4 u more through the fit; nine steps of the fit 3 u; the exponent, at most z^2 + 1.3, rounded at the end and
    twice as 2^(.. log2 e); the exponential 2 u; two products: (18 + 2.5 p^2) u, below 18 (1 + p^2 / 2) u.  Values that end below
    2^-120 may be zero (an exponential that overflows, or whose reciprocal is subnormal).  p comes exactly: one input channel."""
    p = torch.linspace(-13, 13, 15 * M, device=DEV).to(kind).view(15, M)
    for row in p:
        x = torch.zeros(M, 4, device=DEV, dtype=kind)
        x[:, 1] = row
        w = torch.zeros(24, 4, device=DEV, dtype=kind)
        w[:, 1] = 1.0
        got = vq.linear(x, w, None, act)
        assert torch.equal(got, got[:, :1].expand(-1, 24))
        v = row.double()
        if act == "gelu":
            want, each = v * 0.5 * torch.special.erfc(-v / math.sqrt(2)), 18 * (1 + v * v / 2)
        else:
            arg = v if act == "silu" else 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
            want, each = v * torch.sigmoid(arg), 8 + 7 * arg.abs()
        bound = (each * U + (HALF[kind] if kind is not torch.float32 else 0)) * 1.001 * want.abs() + 2.0 ** -120 + TINY[kind]
        seen = (want.abs() > 2.0 ** -100) & (want.abs() > 4 * TINY[kind])
        assert bool((bound < 0.5 * want.abs())[seen].all())      # zero would not pass
        close(got[:, 0], want, bound, act)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_tails_of_the_slopes(act):
    """The same for act'(p) below zero in fp32, where p is kept exactly; s = sigmoid(v) is off by (4 + d) u with v off by d / |v| u.
    silu: s (1 + p (1 - s)), each factor's error and three roundings: 8 s (1 + 2 |p|) u.  gelu: p phi + Phi; phi's exponent p^2 / 2
    is rounded once, and five more: (6 + p^2) |p| phi, Phi's as above, and the last rounding.  gelu_tanh: v rounded five times on
    the way, s + p s (1 - s) v': (10 + 6 |v|) (s + |p| s (1 - s) v') and 1 - s, rounded beside s, 8 |p| v' s^2."""
    p = -torch.linspace(0, 13, 4001, device=DEV)
    x = torch.zeros(4001, 4, device=DEV)
    x[:, 1] = p
    x.requires_grad_()
    w = torch.zeros(1, 4, device=DEV)
    w[:, 1] = 1.0
    (gx,) = torch.autograd.grad(vq.linear(x, w, activation=act), x, torch.ones(4001, 1, device=DEV))
    v = p.double()
    a = v.abs()
    if act == "silu":
        s = torch.sigmoid(v)
        want, bound = s * (1 + v * torch.sigmoid(-v)), 8 * s * (1 + 2 * a)
    elif act == "gelu":
        phi, cdf = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi), 0.5 * torch.special.erfc(-v / math.sqrt(2))
        want = v * phi + cdf
        bound = (6 + v * v) * a * phi + (18 + 9 * v * v) * cdf + want.abs()
    else:
        k = 2 * math.sqrt(2 / math.pi)
        arg, d = k * (v + 0.044715 * v ** 3), k * (1 + 3 * 0.044715 * v * v)
        s, o = torch.sigmoid(arg), torch.sigmoid(-arg)
        want = s + v * s * o * d
        bound = (10 + 6 * arg.abs()) * (s + a * s * o * d) + 8 * a * d * s * s
    bound = bound * U * 1.001 + 2.0 ** -110
    seen = (a > 3) & (want.abs() > 2.0 ** -90)
    assert bool((bound < 0.5 * want.abs())[seen].all())
    close(gx[:, 1], want, bound, act)
    assert not bool(gx[:, [0, 2, 3]].any())


@pytest.mark.parametrize("M", [5, 100])
@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
def test_what_is_kept_for_the_activation(kind, M):
    # fp32, or one rounding to fp16 (half a step 2^-11, 2^-25 near zero) of the product's and the bias's fp32 sum
    from vq_vae_amd import projection
    x, w, b, _, _ = make(M, 96, 130, kind, True, False, False, 31)
    for act in ("silu", "gelu", "gelu_tanh"):
        _, p, _, _, ep = forward64(x, w, b, act, None)
        _, pre = projection.linear_forward(x, w, b, act, want_pre=True)
        assert pre.dtype is (torch.float32 if kind is torch.float32 else torch.float16)
        h, tiny = (0.0, 0.0) if kind is torch.float32 else (2.0 ** -11, 2.0 ** -25)
        close(pre, p, 1.001 * (ep + h * p.abs()) + tiny, act)


@pytest.mark.parametrize("M, K, N", [(1, 2 ** 20, 3), (40, 2 ** 20, 3), (3, 2, 2 ** 20), (33, 2, 2 ** 20)])
def test_the_most_features(M, K, N):
    x, w, b, r, gy = make(M, K, N, torch.bfloat16, True, True, False, 12)
    y, p, slope, ey, ep = forward64(x, w, b, "relu", r)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    out = vq.linear(*leaves, "relu", r)
    close(out.detach(), y, ey, "forward")
    grads = torch.autograd.grad(out, leaves, gy)
    for g, (want, bound), what in zip(grads, backward64(gy, x.detach(), w.detach(), p, ep, slope, "relu"), ("input", "weight", "bias")):
        close(g, want, bound, what)


@pytest.mark.parametrize("M", [3, 40])
def test_rows_far_apart_and_odd_vectors(M):
    # rows further apart than the kernels address are copied first; a bias with gaps and an expanded one too
    K, N = 40, 24
    wide = torch.randn(M, 2 ** 22 + 64, device=DEV).half()
    x, r = wide[:, 5:5 + K], wide[:, 2 ** 22:2 ** 22 + N]
    w = torch.randn(N, 2 ** 22 + 64, device=DEV).half()[:, 3:3 + K]
    for b in (torch.randn(N, 3, device=DEV).half()[:, 1], torch.randn(1, device=DEV).half().expand(N)):
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
        views = [t.detach().requires_grad_() for t in (x, w, b, r)]
        results = []
        for tensors in (leaves, views):
            y = vq.linear(*tensors[:3], "silu", tensors[3])
            results.append([y.detach(), *torch.autograd.grad(y, tensors, torch.ones(M, N, device=DEV, dtype=torch.half))])
        assert all(torch.equal(a, c) for a, c in zip(*results))
