"""The gradient norm and clipping against the formulas in 64 bits.

Tolerances: the norm is summed in 64 bits (errors of 1e-13) and rounded to fp32 once, half a step 2^-24; 2^-23 is allowed.  A
scaled gradient is g times the fp32 factor (half a step of fp32, and 2^-23 for the norm in it), rounded to its type: half a
step of that on top.  Near zero fp16 and bf16 results are off by at most half their smallest step."""
import math

import pytest
import torch

import vq_vae_amd as vq

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def norm64(grads, p=2.0):
    flat = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(1)
    if p == math.inf:
        return float(flat.abs().max()) if flat.numel() else 0.0
    return float(flat.abs().sum()) if p == 1 else float(flat.square().sum().sqrt())


def clipped_ok(out, grads, max_norm, p=2.0):
    c = min(1.0, max_norm / (norm64(grads, p) + 1e-6))
    for o, g in zip(out, grads):
        want = g.double() * c
        bound = want.abs() * (2 * 2.0 ** -23 + HALF[o.dtype]) + TINY[o.dtype]
        assert bool(((o.double() - want).abs() <= bound).all())


def make(sizes, kinds, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * scale).to(kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


# single elements, chunk ends (8192 fp32 or 16384 16-bit elements) on both sides, more tensors than one launch takes
LISTS = {
    "one": [1], "few": [1, 2, 3, 5, 8, 13], "chunk": [8191, 8192, 8193, 16383, 16384, 16385], "large": [3_000_001],
    "many": [7 * i % 1000 + 1 for i in range(400)], "with empty": [0, 5, 0, 0, 70000, 0], "mixed": [1 << 20, 3, 256, 99999, 1, 4096],
}


@pytest.mark.parametrize("kinds", [[t] for t in TYPES] + [TYPES], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
def test_norm_and_clipping(name, kinds):
    for p in (2.0, 1.0, math.inf):
        grads = make(LISTS[name], kinds)
        want = norm64(grads, p)
        got = vq.grad_norm(grads, p)
        assert got.dtype == torch.float32 and got.shape == () and got.device == DEV
        assert abs(float(got) - want) <= 2.0 ** -23 * want
        for max_norm in (0.37 * want, 2 * want + 1, 0.0):
            # into fp32, into the same type, and in place; the sources stay as they were in the first two
            for outs in ([torch.empty_like(g, dtype=torch.float32) for g in grads], [torch.empty_like(g) for g in grads]):
                before = [g.clone() for g in grads]
                n = vq.clip_grads(grads, max_norm, p, out=outs)
                assert float(n) == float(got)
                clipped_ok(outs, grads, max_norm, p)
                assert all(torch.equal(a, b) for a, b in zip(before, grads))
            inplace = [g.clone() for g in grads]
            assert float(vq.clip_grads(inplace, max_norm, p)) == float(got)
            assert all(torch.equal(a, b) for a, b in zip(inplace, outs))


def test_range_of_the_squares():
    # squares outside fp32 and sums beyond its steps
    for scale in (1e30, 1e-30):
        grads = [torch.full((1000,), scale, device=DEV), torch.full((24,), 2 * scale, device=DEV).bfloat16()]
        want = norm64(grads)
        assert abs(float(vq.grad_norm(grads)) - want) <= 2.0 ** -23 * want
    big = torch.ones(1 << 25, device=DEV)
    assert float(vq.grad_norm([big], 1.0)) == 2.0 ** 25
    big[0] = 2.0 ** 24
    assert abs(float(vq.grad_norm([big], 1.0)) - (2 ** 25 + 2 ** 24 - 1)) <= 2.0      # half a step at that size
    # a norm beyond fp32 is infinite, and scales by zero or by what little 64 bits leave
    huge = torch.full((1 << 16,), 3e38, device=DEV)
    assert math.isinf(float(vq.grad_norm([huge])))


@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_nonfinite_gradients(p, bad, kind):
    for where in (0, 40000, 99999):
        grads = make([50, 100_000, 7], [kind])
        grads[1][where] = bad
        norm = float(vq.grad_norm(grads, p))
        assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
        want = [g.float() * (math.nan if math.isnan(bad) else 0.0) for g in grads]      # inf * 0 is NaN, as in the formula
        vq.clip_grads(grads, 1.0, p)
        for g, w in zip(grads, want):
            assert torch.equal(g.isnan(), w.isnan()) and not bool(g[~w.isnan()].any())


def test_clip_grad_norm_of_parameters():
    a = torch.nn.Parameter(torch.zeros(70, 30, device=DEV))
    b = torch.nn.Parameter(torch.zeros(30, device=DEV, dtype=torch.bfloat16))
    c = torch.nn.Parameter(torch.zeros(9, device=DEV))      # without a gradient
    g = make([2100, 30], [torch.float32, torch.bfloat16])
    a.grad, b.grad = g[0].view(70, 30).clone(), g[1].clone()
    n = vq.clip_grad_norm_([a, b, c], 0.5)
    assert abs(float(n) - norm64(g)) <= 2.0 ** -23 * norm64(g)
    clipped_ok([a.grad.view(-1), b.grad], g, 0.5)
    ref = [torch.nn.Parameter(torch.zeros_like(a)), torch.nn.Parameter(torch.zeros_like(b))]
    ref[0].grad, ref[1].grad = g[0].view(70, 30).clone(), g[1].clone()
    torch.nn.utils.clip_grad_norm_(ref[:1], 0.5)
    a.grad = g[0].view(70, 30).clone()
    version = a.grad._version
    vq.clip_grad_norm_(a, 0.5)
    assert a.grad._version > version
    assert float((a.grad - ref[0].grad).abs().max()) <= 4 * 2.0 ** -24 * float(ref[0].grad.abs().max()) + 1e-7 * float(ref[0].grad.abs().max())
    a.grad[0, 0] = math.inf
    before = a.grad.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        vq.clip_grad_norm_([a], 1.0, error_if_nonfinite=True)
    assert torch.equal(a.grad, before)
    a.grad[0, 0] = 1.0
    vq.clip_grad_norm_([a], 1.0, error_if_nonfinite=True)


def test_strides_and_misaligned_views():
    base = torch.randn(400_007, device=DEV)
    views = {
        "offset": lambda: [base.clone()[1:], base.bfloat16()[3:100_000], base.half()[1:2]],
        "transposed": lambda: [torch.randn(300, 500, device=DEV).t()],
        "channels_last": lambda: [torch.randn(4, 40, 9, 11, device=DEV).contiguous(memory_format=torch.channels_last)],
        "columns": lambda: [torch.randn(500, 64, device=DEV)[:, 3:40]],
        "every other": lambda: [torch.randn(9999, device=DEV)[::2], torch.randn(3, device=DEV)],
        "scalar": lambda: [torch.randn((), device=DEV), torch.randn(1, 1, device=DEV)],
    }
    for name, f in views.items():
        grads = f()
        keep = [g.clone() for g in grads]
        want = norm64(keep)
        assert abs(float(vq.grad_norm(grads)) - want) <= 2.0 ** -23 * want, name
        outs = [torch.empty(g.shape, device=DEV) for g in grads]                              # dense, another order than the source
        vq.clip_grads(grads, want / 3, out=outs)
        clipped_ok(outs, keep, want / 3)
        odd = [torch.empty(g.numel(), 2, device=DEV)[:, 0].view(g.shape) if g.dim() == 1 else torch.empty(g.shape, device=DEV) for g in grads]
        vq.clip_grads(grads, want / 3, out=odd)                                               # an output with gaps
        clipped_ok(odd, keep, want / 3)
        vq.clip_grads(grads, want / 3)
        clipped_ok(grads, keep, want / 3)
    # an expanded gradient may be read
    e = torch.randn(5, 1, device=DEV).expand(5, 40)
    assert abs(float(vq.grad_norm([e])) - norm64([e])) <= 2.0 ** -23 * norm64([e])
    outs = [torch.empty(5, 40, device=DEV)]
    vq.clip_grads([e], 0.1, out=outs)
    clipped_ok(outs, [e], 0.1)


def test_neighbours_are_left_alone():
    buf = torch.randn(100_000, device=DEV).bfloat16()
    keep = buf.clone()
    parts = [buf[5:17], buf[17:40_001], buf[50_003:99_990]]
    vq.clip_grads(parts, 0.01)
    for a, b in ((0, 5), (40_001, 50_003), (99_990, 100_000)):
        assert torch.equal(buf[a:b], keep[a:b])
    assert not torch.equal(buf[5:17], keep[5:17])


def test_beyond_two_to_the_31_elements():
    n = 2 ** 31 + 4321
    g = torch.full((n,), 0.5, device=DEV, dtype=torch.bfloat16)
    g[-1] = 512.0
    want = math.sqrt(0.25 * (n - 1) + 512.0 ** 2)
    assert abs(float(vq.grad_norm([g])) - want) <= 2.0 ** -23 * want
    vq.clip_grads([g], want / 2)
    assert float(g[-1]) == 256.0 and float(g[0]) == 0.25 and float(g[2 ** 31]) == 0.25 and float(g[2 ** 30 + 1]) == 0.25
    assert bool((g[:-1].view(-1)[::4097] == 0.25).all())


def test_same_bits_streams_and_graphs():
    sizes = [70001, 5, 300_000, 1] + [64] * 200
    grads = make(sizes, TYPES)
    first = vq.grad_norm(grads)
    assert all(torch.equal(first, vq.grad_norm(grads)) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = vq.grad_norm(grads)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    # two captured passes, replayed in turn on new values between eager work
    held = [make(sizes, TYPES, seed=k) for k in range(2)]
    graphs = []
    for k in range(2):
        outs = [torch.empty(g.shape, device=DEV) for g in held[k]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n = vq.clip_grads(held[k], 2.5, out=outs)
            m = vq.clip_grads(held[k], 1.5)
        graphs.append((graph, outs, n, m))
    for r in range(3):
        for k, (graph, outs, n, m) in enumerate(graphs):
            new = make(sizes, TYPES, seed=20 + 2 * r + k)
            for h, v in zip(held[k], new):
                h.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            want_out = [torch.empty(g.shape, device=DEV) for g in new]
            assert torch.equal(n, vq.clip_grads(new, 2.5, out=want_out))
            assert torch.equal(m, vq.clip_grads(new, 1.5))
            assert all(torch.equal(a, b) for a, b in zip(outs, want_out))
            assert all(torch.equal(a, b) for a, b in zip(held[k], new))


def test_a_training_step():
    """The operators together, as a trainer uses them: projection, hidden layer and its residual, the quantizer, the gradients
    clipped.  Against the formulas in 64 bits with the codes that the quantizer chose."""
    torch.manual_seed(11)
    B, C, H, W, K = 4, 32, 8, 8, 64
    up, down = vq.Linear(C, 4 * C, activation="gelu").to(DEV), vq.Linear(4 * C, C).to(DEV)
    q = vq.EMAVectorQuantizer(K, C, 0.25).to(DEV)
    q.eval()
    h = torch.randn(B, H, W, C, device=DEV)
    t = torch.randn(B, C, H, W, device=DEV)
    z = down(up(h), h)
    out, loss, (_, idx, _) = q(z.permute(0, 3, 1, 2))
    total = ((out - t) ** 2).mean() + loss
    params = [*up.parameters(), *down.parameters()]
    for p in params:
        p.grad = None
    total.backward()
    norm = vq.clip_grad_norm_(params, 0.05)

    ref = [p.detach().double().requires_grad_() for p in params]
    hd = h.double()
    zd = torch.nn.functional.gelu(hd @ ref[0].t() + ref[1]) @ ref[2].t() + ref[3] + hd
    e = q.embedding.weight.detach().double()[idx.view(B, H, W)]
    od = (zd + (e - zd).detach()).permute(0, 3, 1, 2)
    want = ((od - t.double()) ** 2).mean() + 0.25 * ((e.detach() - zd) ** 2).mean()
    grads = torch.autograd.grad(want, ref)
    n = norm64(grads)
    # fp32 throughout: sums of at most 256 terms, relative to the size of each gradient
    assert abs(float(total) - float(want)) <= 1e-5 * abs(float(want))
    assert abs(float(norm) - n) <= 1e-5 * n
    for p, g in zip(params, grads):
        g = g * min(1.0, 0.05 / (n + 1e-6))
        assert float((p.grad.double() - g).abs().max()) <= 2e-5 * float(g.abs().max())


@pytest.mark.parametrize("src, dst", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                      (torch.float32, torch.float32)], ids=["bf16-f32", "f16-f32", "bf16", "f32"])
def test_results_between_others(src, dst):
    # results in the middle of a buffer, at every element offset within 16 bytes, around the sizes of a chunk and of an access
    sizes = [1, 2, 3, 4, 5, 7, 8, 9, 255, 8191, 8192, 8193, 16383, 16384, 16385, 16387, 40003]
    for shift in range(8):
        grads = [torch.randn(n + shift, device=DEV)[shift:].to(src) for n in sizes]
        bufs = [torch.full((n + 64,), 7.0, device=DEV, dtype=dst) for n in sizes]
        outs = [b[16 + shift:16 + shift + n] for b, n in zip(bufs, sizes)]
        norm = vq.clip_grads(grads, 3.0, out=outs)
        want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        assert abs(float(norm) - want) <= 2.0 ** -23 * want
        c = min(1.0, 3.0 / (want + 1e-6))
        for b, o, g, n in zip(bufs, outs, grads, sizes):
            assert bool((b[:16 + shift] == 7).all()) and bool((b[16 + shift + n:] == 7).all())
            h = torch.finfo(dst).eps / 2
            # c in fp32 and a rounding of the product; one of the result
            assert bool(((o.double() - g.double() * c).abs() <= (2.0 ** -22 + 1.01 * h) * g.double().abs() * c + 1e-37).all())


def test_inference_tensors():
    with torch.inference_mode():
        g = [torch.full((5,), 3.0, device=DEV), torch.full((7, 3), 4.0, device=DEV).t()]
        norm = vq.clip_grads(g, 1.0)
    for _ in range(2):      # outside too
        want = math.sqrt(45 + 21 * 16)
        assert abs(float(norm) - want) <= 2.0 ** -22 * want
        assert abs(float(vq.grad_norm(g)) - 1.0) <= 1e-5
        norm = vq.clip_grads([g[0] * want, g[1] * want], 1e9)


@pytest.mark.parametrize("p", [1.0, 2.0])
def test_norms_beyond_fp32_scale_by_zero(p):
    # the norm of finite gradients that fp32 has no number for is infinite, and scales by max_norm / inf; one just inside does not
    n = 1 << 16
    for outs in (False, True):
        g = [torch.full((n,), 3e38, device=DEV), torch.full((9,), -3e38, device=DEV).bfloat16()]
        to = [torch.full((n,), 7.0, device=DEV), torch.full((9,), 7.0, device=DEV)] if outs else g
        assert float(vq.clip_grads(g, 1.0, p, out=to if outs else None)) == math.inf
        assert not any(bool(t.any()) for t in to)
    inside = [torch.full((n,), 1e38 * n ** (-1 / p), device=DEV)]
    keep = [t.clone() for t in inside]
    norm = vq.clip_grads(inside, 1e30, p)
    assert math.isfinite(float(norm))
    clipped_ok(inside, keep, 1e30, p)


def test_max_norms_beyond_fp32():
    # a finite max_norm that fp32 has no number for leaves finite norms alone and is nothing beside an infinite one
    for max_norm in (1e39, 1e300):
        g = make([1000, 7], TYPES)
        keep = [t.clone() for t in g]
        vq.clip_grads(g, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(g, keep))
        g[1][3] = math.inf
        assert float(vq.clip_grads(g, max_norm)) == math.inf
        assert not bool(g[0].any()) and bool(g[1][3].isnan()) and not bool(g[1][:3].any())
    top = torch.full((1,), torch.finfo(torch.float32).max, device=DEV)
    vq.clip_grads([top], 1e39)
    assert float(top) == torch.finfo(torch.float32).max


def test_gradients_that_have_a_graph():
    # as torch's clip_grad_norm_: scaled in place, outside the graph, and known to it as changed
    x = torch.linspace(1, 2, 50, device=DEV).requires_grad_()
    y = x.detach().clone().requires_grad_()
    for v in (x, y):
        (v ** 3).sum().backward(create_graph=True)
    norm = vq.clip_grad_norm_([x], 0.5, error_if_nonfinite=True)
    want = torch.nn.utils.clip_grad_norm_([y], 0.5)
    assert not norm.requires_grad and abs(float(norm) - float(want)) <= 2.0 ** -20 * float(want)
    assert x.grad.grad_fn is not None and float((x.grad - y.grad).abs().max()) <= 2.0 ** -20 * float(y.grad.abs().max())
    (x.grad ** 2).sum()
    with torch.no_grad():
        assert abs(float(vq.grad_norm([x.grad])) - 0.5) <= 1e-6


@pytest.mark.parametrize("kind", TYPES, ids=["f32", "bf16", "f16"])
def test_views_of_one_tensor_that_share_no_element(kind):
    # the gradients of a fused projection's parts, in place, by other views of themselves, and into other columns
    whole = torch.randn(300, 96, device=DEV).to(kind)
    parts = lambda m: [m[:, :31], m[:, 31:64], m[10:, 64:90], m[:10, 64:90:2], m[:10, 65:90:2]]
    for again in (False, True):
        m = whole.clone()
        grads = parts(m)
        keep = [g.clone() for g in grads]
        norm = vq.clip_grads(grads, 3.0, out=parts(m) if again else None)
        want = norm64(keep)
        assert abs(float(norm) - want) <= 2.0 ** -23 * want
        clipped_ok(grads, keep, 3.0)
        assert torch.equal(m[:, 90:], whole[:, 90:])
    m = torch.cat([whole, torch.zeros_like(whole)], 1)
    vq.clip_grads(parts(m), 3.0, out=parts(m[:, 96:]))
    clipped_ok(parts(m[:, 96:]), parts(whole), 3.0)
    assert torch.equal(m[:, :96], whole) and not bool(m[:, 186:].any())


def test_lists_without_an_element():
    for grads in ([torch.zeros(0, device=DEV)], [torch.zeros(3, 0, device=DEV, dtype=t) for t in TYPES] * 60):
        for p in (1.0, 2.0, math.inf):
            assert float(vq.grad_norm(grads, p)) == 0.0
            assert float(vq.clip_grads(grads, 1.0, p)) == 0.0
            assert float(vq.clip_grads(grads, 0.0, p, out=[torch.empty_like(g, dtype=torch.float32) for g in grads])) == 0.0
