"""Workloads of the projection and gradient operators: the matrix product with bias, activation and residual in its
epilogue (forward, and a training pass with all its gradients), the global gradient norm, and clipping by it.

``own`` chooses between the plain torch formulas (32-bit arithmetic, one rounding at the end) and the calls a user makes."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of a prior over codes: a 256-channel row into a hidden layer; latency counts
        linear_case("linear-token", 1, 256, 1024, "bf16", "silu", True, False, False),
        # eight sequences answered together, one token each: the product is bound by reading the weights
        linear_case("linear-decode", 8, 4096, 4096, "bf16", "gelu", True, True, False),
        # an odd batch of latents whose rows are the first half of wider ones (mean and log-variance side by side)
        linear_case("linear-odd", 1237, 251, 517, "f32", "silu", True, True, True),
        # 64 Ki latents of 256 channels (a per-GPU training batch) into a hidden layer
        linear_case("linear-wide", 65536, 256, 1024, "bf16", "gelu_tanh", True, False, False),
        # a large square layer with its residual: bound by the matrix cores
        linear_case("linear-large", 8192, 4096, 4096, "bf16", "none", False, True, False),
        # forward and backward of the hidden layer over the 64 Ki latents of a training batch
        dict(linear_case("train-wide", 65536, 256, 1024, "bf16", "silu", True, False, False), op="train"),
        # the same in single precision with a residual, 16 Ki latents of 512 channels
        dict(linear_case("train-f32", 16384, 512, 512, "f32", "gelu", True, True, False), op="train"),
        # a ragged batch in half precision, strided rows, odd widths
        dict(linear_case("train-odd", 777, 130, 515, "f16", "relu", True, True, True), op="train"),
        # the gradients of two 1x1 convolutions and little else: latency counts
        norm_case("norm-small", "norm", 1, 256, 256, "f32", 1.0),
        # the fp32 gradients of 24 blocks
        norm_case("norm-large", "norm", 24, 1024, 4096, "f32", 1.0),
        # a small odd-sized model, clipped
        norm_case("clip-small", "clip", 3, 131, 517, "f32", 0.5),
        # bf16 matrices and fp32 vectors, clipped into the optimizer's fp32 gradients
        norm_case("clip-large", "clip", 8, 2048, 8192, "mixed", 1.0),
    ]


def linear_case(name, rows, inner, outer, kind, act, bias, residual, strided):
    return {"name": name, "op": "linear", "rows": rows, "inner": inner, "outer": outer, "type": kind, "act": act,
            "bias": bias, "residual": residual, "strided": strided}


def norm_case(name, op, layers, width, hidden, kind, max_norm):
    return {"name": name, "op": op, "layers": layers, "width": width, "hidden": hidden, "type": kind, "max_norm": max_norm}


def draw(rng):
    def log_size(lo, hi, step):
        v = int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
        return max(lo, min(hi, v // step * step))

    op = rng.choice(("linear", "linear", "train", "train", "norm", "clip"))
    if op in ("norm", "clip"):
        width, hidden = log_size(17, 2048, rng.choice((1, 8))), log_size(17, 8192, rng.choice((1, 8)))
        most = max(1, min(48, 200_000_000 // (2 * width * hidden)))
        c = norm_case("", op, rng.randint(1, most), width, hidden, rng.choice(("f32", "bf16", "f16", "mixed")),
                      rng.choice((0.1, 1.0, 1000.0)))
    else:
        step = rng.choice((1, 1, 8, 64))
        kind = rng.choice(("f32", "bf16", "bf16", "f16"))
        inner, outer = log_size(max(16, step), 4096, step), log_size(max(16, step), 4096, step)
        room = (4e9 if kind == "f32" else 1.6e10) / (inner * outer)
        rows = max(1, min(log_size(1, rng.choice((16, 1024, 65536)), 1), int(room)))
        c = linear_case("", rows, inner, outer, kind, rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.5,
                        rng.random() < 0.3)
        c["op"] = op
    del c["name"]
    return c


def shapes_of(case):
    """The parameters of `layers` blocks: two projections with their biases and a gain each."""
    w, h = case["width"], case["hidden"]
    return [(h, w), (h,), (w, h), (w,), (w,)] * case["layers"]


def grad_type(case, shape):
    if case["type"] == "mixed":
        return torch.bfloat16 if len(shape) == 2 else torch.float32
    return TYPES[case["type"]]


# ---------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    dev = torch.device("cuda") if torch.cuda.is_available() else torch.device("cpu")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(shape, scale, kind):
        return torch.randn(shape, generator=gen, device=dev).mul_(scale).to(kind)

    s = {"case": case}
    if case["op"] in ("norm", "clip"):
        # each parameter's gradient has a scale of its own, as layers of different depth have
        s["grads"] = [normal(shape, 10.0 ** (-(i * 7 % 5)), grad_type(case, shape)) for i, shape in enumerate(shapes_of(case))]
        if case["op"] == "clip":
            s["out"] = [torch.empty(g.shape, dtype=torch.float32, device=dev) for g in s["grads"]]
        return s
    M, K, N, kind = case["rows"], case["inner"], case["outer"], TYPES[case["type"]]
    x = normal((M, 2 * K), 1.0, kind)[:, :K] if case["strided"] else normal((M, K), 1.0, kind)
    s["x"] = x
    s["weight"] = normal((N, K), K ** -0.5, kind)
    s["bias"] = normal((N,), 0.5, kind) if case["bias"] else None
    s["residual"] = normal((M, N), 1.0, kind) if case["residual"] else None
    if case["op"] == "train":
        s["grad"] = normal((M, N), 0.05, kind)
        s["leaves"] = [t.requires_grad_() for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        import vq_vae_amd as vq
        if case["op"] == "norm":
            return vq.grad_norm(state["grads"])
        if case["op"] == "clip":
            norm = vq.clip_grads(state["grads"], case["max_norm"], out=state["out"])
            return {"norm": norm, "grads": state["out"]}
        y = vq.linear(state["x"], state["weight"], state["bias"], activation=case["act"], residual=state["residual"])
        if case["op"] == "linear":
            return y
        return {"y": y.detach(), "grads": list(torch.autograd.grad(y, state["leaves"], state["grad"]))}
    with torch.no_grad():
        if case["op"] == "norm":
            return plain_norm(state["grads"])
        if case["op"] == "clip":
            norm = plain_norm(state["grads"])
            scale = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
            return {"norm": norm, "grads": [o.copy_(g.float() * scale) for g, o in zip(state["grads"], state["out"])]}
        return plain_linear(state, case)


def plain_norm(grads):
    squares = [g.float().square().sum(dtype=torch.float64) for g in grads]
    return torch.stack(squares).sum().sqrt().float()


def plain_linear(state, case):
    kind = state["x"].dtype
    x, w = state["x"].float(), state["weight"].float()
    p = x @ w.t()
    if state["bias"] is not None:
        p = p + state["bias"].float()
    a, slope = plain_act(p, case["act"], case["op"] == "train")
    y = a if state["residual"] is None else a + state["residual"].float()
    y = y.to(kind)
    if case["op"] == "linear":
        return y
    gy = state["grad"].float()
    dp = gy if slope is None else gy * slope
    grads = [(dp @ w).to(kind), (dp.t() @ x).to(kind)]
    if state["bias"] is not None:
        grads.append(dp.sum(0).to(kind))
    if state["residual"] is not None:
        grads.append(state["grad"])
    return {"y": y, "grads": grads}


def plain_act(p, act, want_slope):
    """act(p) and, where it is wanted, its derivative."""
    if act == "none":
        return p, None
    if act == "relu":
        return p.clamp(min=0), (p > 0).float() if want_slope else None
    if act == "silu":
        s = 1 / (1 + torch.exp(-p))
        return p * s, s * (1 + p * (1 - s)) if want_slope else None
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(p * 0.5 ** 0.5))
        return p * cdf, cdf + p * torch.exp(-0.5 * p * p) * (2 * math.pi) ** -0.5 if want_slope else None
    c = (2 / math.pi) ** 0.5
    t = torch.tanh(c * (p + 0.044715 * p * p * p))
    slope = 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p) if want_slope else None
    return 0.5 * p * (1 + t), slope


# ---------------------------------------------------------------------------------------------------- the work
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "mixed": 2}
    if case["op"] in ("norm", "clip"):
        shapes = shapes_of(case)
        read = sum(math.prod(s) * grad_type(case, s).itemsize for s in shapes)
        count = sum(math.prod(s) for s in shapes)
        write = 4 * count if case["op"] == "clip" else 0
        return {"bytes": read + write + 4, "flops": (3 if case["op"] == "clip" else 2) * count}
    M, K, N, t = case["rows"], case["inner"], case["outer"], size[case["type"]]
    ends = M * K + N * K + (N if case["bias"] else 0)          # x, weight, bias: read, and in training their gradients written
    if case["op"] == "linear":
        return {"bytes": t * (ends + M * N * (2 if case["residual"] else 1)), "flops": 2 * M * N * K}
    return {"bytes": t * (2 * ends + M * N * (3 if case["residual"] else 2)), "flops": 6 * M * N * K}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "clip"):
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
        as_tensor = torch.tensor(norm, dtype=torch.float64, device=s["grads"][0].device)
        if case["op"] == "norm":
            return as_tensor
        c = min(1.0, case["max_norm"] / (norm + 1e-6))
        return {"norm": as_tensor, "grads": [g.double() * c for g in s["grads"]]}
    F = torch.nn.functional
    act = {"none": lambda v: v, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}
    wide = {k: s[k].detach().double().requires_grad_() for k in ("x", "weight", "bias", "residual") if s[k] is not None}
    y = act[case["act"]](F.linear(wide["x"], wide["weight"], wide.get("bias")))
    if "residual" in wide:
        y = y + wide["residual"]
    if case["op"] == "linear":
        return y.detach()
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, list(wide.values()), s["grad"].double()))}
