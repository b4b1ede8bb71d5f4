"""What is timed of a pre-norm gated encoder block's operators, beside the plain forms of the same.

Kinds of cases
  norm     residual add + root-mean-square norm: forward and backward ("train"), forward ("infer"), forward with an output in
           8 bits and a scale per row ("8bit")
  gated    act(x Wg^T + bg) * (x Wu^T + bu): forward and backward, forward, forward on operands in 8 bits
  linear   act(x W^T + b) + residual: the same three

Inputs are synthetic, made on the GPU from the seed alone: a residual stream with some loud features, weights of the scale
1 / sqrt(width), gradients of order one.
"""
import math
import types

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # one new row of a wide model: launch latency alone
        {"name": "norm_1x1024_bf16", "kind": "norm", "mode": "infer", "rows": 1, "width": 1024, "residual": True, "dtype": "bf16"},
        # a training step's norm at the headline graph: one sequence of 64 000 nodes, hidden 64, float32
        {"name": "norm_64000x64_f32", "kind": "norm", "mode": "train", "rows": 64000, "width": 64, "residual": True, "dtype": "f32"},
        # the same of a wide model, 16 K rows of 2048 features
        {"name": "norm_16384x2048_bf16", "kind": "norm", "mode": "train", "rows": 16384, "width": 2048, "residual": True,
         "dtype": "bf16"},
        # the norm in front of a product in 8 bits, a ragged number of rows
        {"name": "norm_8bit_8191x1408_bf16", "kind": "norm", "mode": "8bit", "rows": 8191, "width": 1408, "residual": True,
         "dtype": "bf16"},
        # one new row through the gated projections: the weights' bytes count
        {"name": "gated_1x1024x4096_bf16", "kind": "gated", "mode": "infer", "rows": 1, "width": 1024, "hidden": 4096,
         "act": "silu", "bias": False, "dtype": "bf16"},
        # a training step's gated projections at the headline graph, hidden 64, ffn 128, float32
        {"name": "gated_64000x64x128_f32", "kind": "gated", "mode": "train", "rows": 64000, "width": 64, "hidden": 128,
         "act": "gelu", "bias": True, "dtype": "f32"},
        # a training step of a wide model
        {"name": "gated_16384x1024x4096_bf16", "kind": "gated", "mode": "train", "rows": 16384, "width": 1024, "hidden": 4096,
         "act": "silu", "bias": False, "dtype": "bf16"},
        # serving in 8 bits, a ragged batch
        {"name": "gated_8bit_4099x1024x2816", "kind": "gated", "mode": "8bit", "rows": 4099, "width": 1024, "hidden": 2816,
         "act": "silu", "bias": False, "dtype": "bf16"},
        # the projection back to the residual stream for seven new rows
        {"name": "linear_7x4096x1024_bf16", "kind": "linear", "mode": "infer", "rows": 7, "width": 4096, "hidden": 1024,
         "act": "none", "bias": True, "residual": True, "dtype": "bf16"},
        # a training step with odd widths, float32: 37 605 nodes (the ragged last part of an epoch), 100 features to 47
        {"name": "linear_37605x100x47_f32", "kind": "linear", "mode": "train", "rows": 37605, "width": 100, "hidden": 47,
         "act": "gelu", "bias": True, "residual": False, "dtype": "f32"},
        # a training step's projection back to the residual stream of a wide model
        {"name": "linear_16384x4096x1024_bf16", "kind": "linear", "mode": "train", "rows": 16384, "width": 4096, "hidden": 1024,
         "act": "none", "bias": True, "residual": True, "dtype": "bf16"},
        # queries, keys and values of a ragged batch in 8 bits, in one product
        {"name": "linear_8bit_2050x2048x6144", "kind": "linear", "mode": "8bit", "rows": 2050, "width": 2048, "hidden": 6144,
         "act": "none", "bias": True, "residual": False, "dtype": "bf16"},
    ]


MOST_FLOPS = 12.0 * 16384 * 1024 * 4096      # of the largest listed case, a training step of the gated projections
MOST_VALUES = 16384 * 2048                   # of a norm


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths as models have them: most a multiple of 64 or 8, some odd."""
    w = _log(rng, lo, hi)
    step = rng.choice([64, 64, 8, 1])
    return max(step, w // step * step)


def draw(rng):
    kind = rng.choice(["norm", "gated", "linear"])
    mode = rng.choice(["train", "train", "infer", "8bit"])
    dtype = "bf16" if mode == "8bit" else rng.choice(["f32", "bf16"])
    rows = _log(rng, 1, 64) if mode == "infer" else _log(rng, 200, 64000)
    if kind == "norm":
        width = _width(rng, 64, 4096)
        return {"kind": kind, "mode": mode, "rows": min(rows, MOST_VALUES // width), "width": width,
                "residual": rng.random() < 0.8, "dtype": dtype}
    # the plain forms are products in 32 bits on both sides: float32 keeps to the widths of this framework's models
    wide = 512 if dtype == "f32" else 4096
    width, hidden = _width(rng, 64, wide), _width(rng, 47, wide)
    if mode == "8bit":
        width = max(16, width // 16 * 16)
    rows = max(1, min(rows, int(MOST_FLOPS / (12.0 * width * hidden))))
    case = {"kind": kind, "mode": mode, "rows": rows, "width": width, "hidden": hidden, "bias": rng.random() < 0.5, "dtype": dtype}
    if kind == "gated":
        case["act"] = rng.choice(["silu", "gelu", "relu"])
    else:
        case["act"] = rng.choice(["none", "none", "gelu", "relu", "silu"])
        case["residual"] = rng.random() < 0.5
    return case


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _loud(g, width):
    """Features of a residual stream differ in size: one in sixty-four is ten times as loud."""
    return torch.where(torch.rand(width, generator=g, device=DEV) < 1.0 / 64, 10.0, 1.0)


def _codes(t):
    """A matrix in 8 bits with a scale per row, as a program keeps its weights and the norm hands over its rows.  A row's scale is
    the smallest power of two that brings its largest value to at most 448: the codes have an exponent of their own, so a finer
    scale would gain nothing, and a power of two neither rounds nor puts values on the borders between codes."""
    m, e = torch.frexp(t.abs().amax(dim=1))
    scales = torch.ldexp(torch.ones_like(m), torch.where(m > 0.875, e - 8, e - 9))
    return (t / scales[:, None]).to(E4M3), scales


def _values(codes, scales):
    """What the codes stand for: a power of two times four bits is exact in bfloat16."""
    return (codes.float() * scales[:, None]).to(torch.bfloat16)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, N, C = DTYPES[case["dtype"]], case["rows"], case["width"]
    s = types.SimpleNamespace(case=case)
    if case["kind"] == "norm":
        loud = _loud(g, C)
        s.x = (_normal(g, N, C) * loud).to(dt)
        s.r = _normal(g, N, C).to(dt) if case["residual"] else None
        s.w = (1.0 + _normal(g, C, scale=0.2)).to(dt)
        if case["mode"] == "train":
            s.dy, s.ds = _normal(g, N, C).to(dt), _normal(g, N, C).to(dt)
        return s
    M = case["hidden"]
    x = _normal(g, N, C)
    names = ("wg", "wu") if case["kind"] == "gated" else ("w",)
    for name in names:
        w = _normal(g, M, C, scale=1.5 / math.sqrt(C))
        if case["mode"] == "8bit":
            codes, scales = _codes(w)
            setattr(s, name, codes)
            setattr(s, name + "_scales", scales)
        else:
            setattr(s, name, w.to(dt))
    for name in ("bg", "bu") if case["kind"] == "gated" else ("b",):
        setattr(s, name, _normal(g, M, scale=0.1).to(dt) if case["bias"] else None)
    if case["mode"] == "8bit":
        s.x, s.x_scales = _codes(x * _loud(g, C))
    else:
        s.x = x.to(dt)
    s.r = _normal(g, N, M).to(dt) if case.get("residual") else None
    if case["mode"] == "train":
        s.dy = _normal(g, N, M).to(dt)
    return s


LEAVES = {"norm": ("x", "r", "w"), "gated": ("x", "wg", "wu", "bg", "bu"), "linear": ("x", "w", "b", "r")}


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["mode"] == "train":
        s.leaves = [getattr(s, n).requires_grad_(True) for n in LEAVES[case["kind"]] if getattr(s, n) is not None]
    return s


def run(s):
    return (_own if own else _plain)(s)


# ---- the framework's operators ------------------------------------------------------------------------------------------------

def _own(s):
    import torchgt_amd as T
    case = s.case
    kind, mode = case["kind"], case["mode"]
    act = None if case.get("act") == "none" else case.get("act")
    if kind == "norm":
        if mode == "8bit":
            total, codes, scales = T.add_rms_norm_8bit(s.x, s.r, s.w, EPS)
            return [total, _values(codes, scales), scales]
        if mode == "infer":
            return list(T.add_rms_norm(s.x, s.r, s.w, EPS))
        total, y = T.add_rms_norm(s.x, s.r, s.w, EPS)
        return [total.detach(), y.detach()] + list(torch.autograd.grad((total, y), s.leaves, (s.ds, s.dy)))
    if kind == "gated":
        if mode == "8bit":
            return T.gated_linear_8bit(s.x, s.x_scales, s.wg, s.wg_scales, s.wu, s.wu_scales, s.bg, s.bu, activation=act)
        y = T.gated_linear(s.x, s.wg, s.wu, s.bg, s.bu, activation=act)
    else:
        if mode == "8bit":
            return T.linear_act_8bit(s.x, s.x_scales, s.w, s.w_scales, s.b, activation=act, residual=s.r)
        y = T.linear_act(s.x, s.w, s.b, activation=act, residual=s.r)
    if mode == "infer":
        return y
    return [y.detach()] + list(torch.autograd.grad(y, s.leaves, s.dy))


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ---------------------------------------------------

def _act(name, u):
    if name == "silu":
        return u * torch.sigmoid(u)
    if name == "gelu":
        return 0.5 * u * (1.0 + torch.erf(u * math.sqrt(0.5)))
    return torch.where(u > 0, u, torch.zeros_like(u)) if name == "relu" else u


def _slope(name, u):
    if name == "silu":
        e = torch.sigmoid(u)
        return e * (1.0 + u * (1.0 - e))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2.0 * math.pi)
    return (u > 0).to(u.dtype) if name == "relu" else torch.ones_like(u)


def _plain(s):
    with torch.no_grad():
        return {"norm": _plain_norm, "gated": _plain_gated, "linear": _plain_linear}[s.case["kind"]](s)


def _wide(t, scales=None):
    if t is None:
        return None
    return t.float() if scales is None else t.float() * scales[:, None]


def _plain_norm(s):
    mode, dt = s.case["mode"], s.x.dtype
    x, w = s.x.float(), s.w.float()
    # the sum is handed on in its type, and the norm is the norm of what is handed on
    total = (x + s.r.float()).to(dt) if s.r is not None else s.x.detach()
    t = total.float()
    rstd = torch.rsqrt((t * t).mean(dim=1, keepdim=True) + EPS)
    xhat = t * rstd
    y = xhat * w
    if mode == "8bit":
        codes, scales = _codes(y)
        return [total, _values(codes, scales), scales]
    if mode == "infer":
        return [total, y.to(dt)]
    dy = s.dy.float()
    g = dy * w
    dt_total = ((g - xhat * (g * xhat).mean(dim=1, keepdim=True)) * rstd + s.ds.float()).to(dt)
    dw = (dy * xhat).sum(dim=0).to(dt)
    return [total, y.to(dt), dt_total] + ([dt_total] if s.r is not None else []) + [dw]


def _plain_gated(s):
    mode, act = s.case["mode"], s.case["act"]
    dt = DTYPES[s.case["dtype"]]
    if mode == "8bit":
        x, wg, wu = _wide(s.x, s.x_scales), _wide(s.wg, s.wg_scales), _wide(s.wu, s.wu_scales)
    else:
        x, wg, wu = _wide(s.x), _wide(s.wg), _wide(s.wu)
    g, u = x @ wg.t(), x @ wu.t()
    if s.bg is not None:
        g, u = g + s.bg.float(), u + s.bu.float()
    h = (_act(act, g) * u).to(dt)
    if mode != "train":
        return h
    dh = s.dy.float()
    dg, du = dh * u * _slope(act, g), dh * _act(act, g)
    out = [h, (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)]
    return out + ([dg.sum(dim=0).to(dt), du.sum(dim=0).to(dt)] if s.bg is not None else [])


def _plain_linear(s):
    mode, act = s.case["mode"], s.case["act"]
    dt = DTYPES[s.case["dtype"]]
    if mode == "8bit":
        x, w = _wide(s.x, s.x_scales), _wide(s.w, s.w_scales)
    else:
        x, w = _wide(s.x), _wide(s.w)
    u = x @ w.t()
    if s.b is not None:
        u = u + s.b.float()
    y = _act(act, u)
    if s.r is not None:
        y = y + s.r.float()
    y = y.to(dt)
    if mode != "train":
        return y
    du = s.dy.float() * _slope(act, u)
    out = [y, (du @ w).to(dt), (du.t() @ x).to(dt)]
    return out + ([du.sum(dim=0).to(dt)] if s.b is not None else []) + ([s.dy] if s.r is not None else [])


# ---- bytes and operations of one pass ----------------------------------------------------------------------------------------------

def work(case):
    e, N, C, train = (4 if case["dtype"] == "f32" else 2), case["rows"], case["width"], case["mode"] == "train"
    if case["kind"] == "norm":
        r = 1 if case["residual"] else 0
        if case["mode"] == "8bit":
            return {"bytes": N * C * ((1 + 2 * r) * e + 1) + C * e + 4 * N, "flops": 8.0 * N * C}
        # forward: x (and r) in, y (and the sum) out; backward: two gradients in, one out
        return {"bytes": N * C * e * (2 + 2 * r + (3 if train else 0)) + C * e * (2 if train else 1), "flops": (16.0 if train else 5.0) * N * C}
    M, n = case["hidden"], (2 if case["kind"] == "gated" else 1)
    ei = 1 if case["mode"] == "8bit" else e
    read = N * C * ei + n * M * C * ei + (n * M * e if case["bias"] else 0)
    if case["mode"] == "8bit":
        read += 4 * (N + n * M)
    size = read + N * M * e * (2 if case.get("residual") else 1)
    if train:      # the gradient of the output in, those of x, the weights and biases out
        size += N * M * e + N * C * e + n * M * C * e + (n * M * e if case["bias"] else 0)
    return {"bytes": size, "flops": 2.0 * n * N * C * M * (3 if train else 1)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------

def _erf_gelu(z):
    return z / 2 * torch.special.erfc(-z / math.sqrt(2))


CURVES = {
    "silu": (lambda z: z / (1 + torch.exp(-z)), lambda z: 1 / (1 + torch.exp(-z)) + z * torch.exp(-z.abs()) / (1 + torch.exp(-z.abs())) ** 2),
    "gelu": (_erf_gelu, lambda z: torch.special.erfc(-z / math.sqrt(2)) / 2 + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
    "relu": (lambda z: z.clamp(min=0), lambda z: (z > 0).double()),
    "none": (lambda z: z, lambda z: torch.ones_like(z)),
}


def exact(case, seed):
    s = _inputs(case, seed)
    d = lambda t: None if t is None else t.double()      # noqa: E731
    if case["kind"] == "norm":
        return _exact_norm(case, s, d)
    deq = (lambda n: getattr(s, n).double() * getattr(s, n + "_scales").double().unsqueeze(1)) if case["mode"] == "8bit" else (lambda n: d(getattr(s, n)))
    f, slope = CURVES[case["act"]]
    x = deq("x")
    if case["kind"] == "gated":
        wg, wu = deq("wg"), deq("wu")
        a, b = torch.mm(x, wg.T), torch.mm(x, wu.T)
        if case["bias"]:
            a, b = a + d(s.bg), b + d(s.bu)
        h = f(a) * b
        if case["mode"] != "train":
            return h
        ga, gb = slope(a) * b * d(s.dy), f(a) * d(s.dy)
        grads = [torch.mm(ga, wg) + torch.mm(gb, wu), torch.mm(ga.T, x), torch.mm(gb.T, x)]
        return [h] + grads + ([ga.sum(0), gb.sum(0)] if case["bias"] else [])
    w = deq("w")
    a = torch.mm(x, w.T)
    if case["bias"]:
        a = a + d(s.b)
    y = f(a) + (d(s.r) if case["residual"] else 0.0)
    if case["mode"] != "train":
        return y
    ga = slope(a) * d(s.dy)
    return [y, torch.mm(ga, w), torch.mm(ga.T, x)] + ([ga.sum(0)] if case["bias"] else []) + ([d(s.dy)] if case["residual"] else [])


def _exact_norm(case, s, d):
    # the definition takes the norm of the sum as it is stored
    total = d(s.x if s.r is None else (d(s.x) + d(s.r)).to(s.x.dtype))
    size = torch.sqrt(total.square().sum(1, keepdim=True) / case["width"] + EPS)
    unit = total / size
    y = unit * d(s.w)
    kept = total if s.r is None else d(s.x) + d(s.r)
    if case["mode"] == "8bit":
        unit_size = torch.exp2(torch.ceil(torch.log2(y.abs().max(dim=1, keepdim=True).values / 448.0)))
        # nearest of the 8-bit values, ties to the even one: steps of an eighth of the power of two below, of 2^-9 under 2^-6
        z = y / unit_size
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        return [kept, torch.round(z / step) * step * unit_size, unit_size[:, 0]]
    if case["mode"] == "infer":
        return [kept, y]
    dy = d(s.dy)
    along = (dy * y).sum(1, keepdim=True) / case["width"]
    grad = (dy * d(s.w) - unit * along) / size + d(s.ds)
    return [kept, y, grad] + ([grad] if s.r is not None else []) + [(dy * unit).sum(0)]
