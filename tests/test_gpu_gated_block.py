"""The operators of a pre-norm gated block against their formulas in 64 bits.

Every bound is a sum of what the arithmetic may lose, element by element:
  * a float32 sum of n terms: n 2^-23 of the sum of their magnitudes (the matrix instructions may cut instead of rounding; float32 operands in three
    parts leave out less than 2^-23 of a product: two more terms' worth);
  * a rounding to the tensors' type: eps / 2 of the value;
  * where a forward keeps g and u for its backward (`kept`: float32 from 128 features on, bfloat16 from 512, where the kernels for small widths do not
    take the call): their rounding, in the gradients;
  * a function value: 2^-20 of the largest magnitude that goes into it (erff and expf are good to a few units of 2^-24), bfloat16 results 2^-14
    (v_exp_f32 of a product rounded to 24 bits);
  * operands in 8 bits: the matrix instruction adds eight neighbouring products at a time, aligned to the largest of them and cut 13 binary places below it
    (seen from sums of powers of two: beside a product of 2^12 one of 2^-1 counts and one of 2^-2 does not if it is among the same eight, and does down
    to 2^-11 in any other place): less than 2^-13 of the largest for each of eight, 2^-10 of the largest of every eight;
and what those errors do downstream by the first-order rule, slopes bounded by 1.13 (gelu, silu) and curvatures by 0.8.
"""
import math

import pytest
import torch

import torchgt_amd as T
from torchgt_amd import _lib

pytestmark = pytest.mark.gpu

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
EPS = 1e-6


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rand(g, *shape, dt=F32, scale=1.0, device="cuda"):
    return (torch.randn(*shape, generator=g) * scale).to(dt).to(device)


def act64(name, u):
    if name == "silu":
        return u * torch.sigmoid(u)
    if name == "gelu":
        return 0.5 * u * torch.special.erfc(-u / math.sqrt(2))
    return u.clamp(min=0) if name == "relu" else u


def slope64(name, u):
    if name == "silu":
        s = torch.sigmoid(u)
        return s * (1 + u * (1 - s))
    if name == "gelu":
        return 0.5 * torch.special.erfc(-u / math.sqrt(2)) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    return (u > 0).double() if name == "relu" else torch.ones_like(u)


def curve(name, u, eu, edge=None):
    """How much the slope may be off for an argument off by eu (its sign sure from `edge` on)."""
    if name in ("silu", "gelu"):
        return 0.8 * eu
    return (u.abs() <= (eu if edge is None else edge)).double() if name == "relu" else torch.zeros_like(u)


def fine(dt):
    return 2.0 ** -20 if dt == F32 else 2.0 ** -14


def sums(n):
    return (n + 8) * 2.0 ** -23


class Mapped:
    """value and error bound of one float32 product a b^T (+ bias), from exact operands"""

    def __init__(self, a, b, bias=None, ea=None, eb=None, eight=False):
        self.v = a @ b.T
        m = a.abs() @ b.abs().T
        self.e = sums(a.shape[1]) * m
        if eight:
            for k in range(0, a.shape[1], 8):
                self.e = self.e + 2.0 ** -10 * (a[:, None, k:k + 8] * b[None, :, k:k + 8]).abs().amax(2)
        if ea is not None:
            self.e = self.e + ea @ b.abs().T * (1 + sums(a.shape[1]))
        if eb is not None:
            self.e = self.e + a.abs() @ eb.T * (1 + sums(a.shape[1]))
        if bias is not None:
            self.v = self.v + bias
            self.e = self.e + 2.0 ** -23 * (m + bias.abs())


def stored(v, e, dt):
    return half_step(dt) * (v.abs() + e) + e + 1e-30


def near(got, v, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == v.shape, (what, got.shape, v.shape)
    off = (got - v).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / bound).nan_to_num(1e9).max()):.3g} of its bound, at {bad.nonzero()[0].tolist()}"


def d(t):
    return None if t is None else t.detach().double().cpu()


# ---- gated projections ---------------------------------------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (16, 256, 64), (17, 100, 47), (33, 40, 129), (130, 64, 128), (257, 96, 40), (300, 131, 70), (129, 520, 264),
          (1000, 64, 96), (2049, 72, 130), (5, 1024, 300)]


def gated_case(N, K, F, dt, act, bias, seed=0):
    g = torch.Generator().manual_seed(seed + N * 7 + K * 3 + F)
    x = rand(g, N, K, dt=dt)
    wg, wu = (rand(g, F, K, dt=dt, scale=1.2 / math.sqrt(K)) for _ in range(2))
    bg, bu = (rand(g, F, dt=dt, scale=0.3) if bias else None for _ in range(2))
    return x, wg, wu, bg, bu, rand(g, N, F, dt=dt)


class Kept:
    """A value with its error bound as a backward reads what the forward kept: float32 (or a sign: `edge` is how far from zero it is sure), or four columns of 14 bits at the exponent of the largest (a step is at most
    2^-12 of the largest, and the last step below the next exponent is cut, not rounded: off by half a step, 2^-13, in either case: 8191.5 to 8192 of them
    become 8191, less than one step of 2^-13 of at least 8191.5 of them;
    for a relu those that would round to zero become a step)"""

    def __init__(self, m, dt):
        self.v, self.e, self.edge = m.v, m.e, m.e
        if dt == BF16:
            N, F = m.v.shape
            most = torch.nn.functional.pad(m.v.abs() + m.e, (0, -F % 4)).view(N, -1, 4).amax(2).repeat_interleave(4, 1)[:, :F]
            self.e = m.e + 1.01 * 2.0 ** -12 * most


def check_gated(x, wg, wu, bg, bu, dh, act, outs, kept=False):
    dt = x.dtype
    X, WG, WU, BG, BU, DH = d(x), d(wg), d(wu), d(bg), d(bu), d(dh)
    g, u = Mapped(X, WG, BG), Mapped(X, WU, BU)
    a = act64(act, g.v)
    ea = 1.13 * g.e + fine(dt) * (g.v.abs() + g.e)
    h = a * u.v
    eh = ea * (u.v.abs() + u.e) + a.abs() * u.e + 2.0 ** -23 * h.abs()
    near(outs["h"], h, stored(h, eh, dt), "h")
    if dh is None:
        return
    if kept:
        g, u = Kept(g, dt), Kept(u, dt)
        ea = 1.13 * g.e + fine(dt) * (g.v.abs() + g.e)
    s = slope64(act, g.v)
    es = curve(act, g.v, g.e, getattr(g, "edge", None)) + fine(dt) * (1 + g.v.abs())
    dg, du = DH * u.v * s, DH * a
    edg = DH.abs() * (u.v.abs() * es + (s.abs() + es) * u.e) + 2.0 ** -22 * dg.abs()
    edu = DH.abs() * ea + 2.0 ** -22 * du.abs()
    edg, edu = stored(dg, edg, dt), stored(du, edu, dt)
    both, eboth, W = torch.cat([dg, du], 1), torch.cat([edg, edu], 1), torch.cat([WG, WU], 0)
    dx = Mapped(both, W.T, ea=eboth)
    near(outs["x"], dx.v, stored(dx.v, dx.e, dt), "dx")
    F = wg.shape[0]
    dw = Mapped(both.T, X.T, ea=eboth.T)
    near(outs["wg"], dw.v[:F], stored(dw.v, dw.e, dt)[:F], "dWg")
    near(outs["wu"], dw.v[F:], stored(dw.v, dw.e, dt)[F:], "dWu")
    if bg is not None:
        db, edb = both.sum(0), eboth.sum(0) + sums(len(X)) * both.abs().sum(0)
        near(outs["bg"], db[:F], stored(db, edb, dt)[:F], "dbg")
        near(outs["bu"], db[F:], stored(db, edb, dt)[F:], "dbu")


def run_gated(x, wg, wu, bg, bu, dh, act):
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in dict(x=x, wg=wg, wu=wu, bg=bg, bu=bu).items() if v is not None}
    h = T.gated_linear(leaves["x"], leaves["wg"], leaves["wu"], leaves.get("bg"), leaves.get("bu"), activation=act)
    grads = torch.autograd.grad(h, list(leaves.values()), dh)
    return {"h": h, **dict(zip(leaves, grads))}


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True)])
def test_gated_linear(cuda, shape, dt, act, bias):
    case = gated_case(*shape, dt, act, bias)
    check_gated(*case, act, run_gated(*case, act))


# Beyond the kernels for small widths: tiles of 128, what the forward keeps; whole rows, odd contractions, odd results
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", [(300, 600, 900), (100, 1031, 520), (131, 640, 901), (65, 1040, 1024)])
def test_wider_ones(cuda, shape, dt):
    L, (N, K, F) = _lib.lib(), shape
    code = _lib.DTYPE_F32 if dt == F32 else _lib.DTYPE_BF16
    size = torch.finfo(dt).bits // 8
    room = N * (F if dt == F32 else (F + 3) // 4 * 4) * size
    assert L.tgt_gated_linear_kept_bytes(N, K, F, code, 3) == 2 * room
    case = gated_case(*shape, dt, "silu", True)
    for act in ("silu", "relu"):
        check_gated(*case, act, run_gated(*case, act), kept=True)
    kept = L.tgt_linear_epilogue_kept_bytes(N, K, F, code, 1)
    assert kept in (0, room) and L.tgt_linear_epilogue_kept_bytes(N, K, F, code, 0) == 0
    case = linear_case(*shape, dt, True, True)
    for act in ("gelu", "relu"):
        check_linear(*case, act, run_linear(*case, act), kept=kept > 0)
    check_linear(*case, None, run_linear(*case, None))
    with torch.no_grad():
        x, w, b, r, _ = case
        check_linear(x, w, b, r, None, "relu", {"y": T.linear_act(x, w, b, "relu", r)})


# Small widths and many nodes: the kernels that hold a weight's columns, at the largest weights that they are given
@pytest.mark.parametrize("shape", [(4100, 512, 512), (4097, 68, 1000), (16400, 1024, 60)])
def test_small_widths_many_rows(cuda, shape):
    N, K, F = shape
    case = gated_case(N, K, F // 2, F32, "silu", True)
    check_gated(*case, "silu", run_gated(*case, "silu"))
    case = linear_case(N, K, F, F32, True, True)
    for act in (None, "gelu"):
        check_linear(*case, act, run_linear(*case, act))


# Few tiles and a long contraction, cut in pieces whose sums are joined: rows and columns that end inside a tile or a piece of one, contractions that end inside
# a step and that change from one weight to the other inside and at the border of a piece, operands at odd addresses
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", [(65, 1536, 712), (300, 2048, 264), (257, 1100, 264), (129, 520, 1536), (70, 264, 2048), (513, 1031, 1029)])
def test_contractions_in_pieces(cuda, shape, dt):
    N, K, F = shape
    case = gated_case(N, K, F, dt, "silu", True)
    kept = _lib.lib().tgt_gated_linear_kept_bytes(N, K, F, _lib.DTYPE_F32 if dt == F32 else _lib.DTYPE_BF16, 3)
    check_gated(*case, "silu", run_gated(*case, "silu"), kept=kept > 0)
    case = linear_case(N, K, F, dt, True, True)
    check_linear(*case, None, run_linear(*case, None))
    x, w, b, r, _ = case
    wide = torch.empty(F * K + 1, device="cuda", dtype=dt)
    odd = wide[1:].view(F, K)
    odd.copy_(w)
    with torch.no_grad():
        for weight in (w, odd):
            check_linear(x, w, b, r, None, "gelu", {"y": T.linear_act(x, weight, b, "gelu", r)})


def unpacked(t):
    """Four values in eight bytes, as the backward reads them"""
    n = t.contiguous().view(torch.int64).cpu()
    e = n >> 56 & 255
    m = torch.stack([n >> 14 * i & 0x3fff for i in range(4)], 2)
    v = torch.ldexp((m - (m >> 13) * 16384).double(), (e - 139)[..., None])
    own = torch.from_numpy((m << 18).numpy().astype("uint32").view("float32")).double()
    return torch.where((e == 255)[..., None], own, v).flatten(1)


def test_kept_values_of_any_size(cuda):
    """bfloat16: tiny, huge and infinite products beside others, kept and read back."""
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    row = torch.tensor([1.0, -1.99, 0.5, 2.0 ** -10, 2.0 ** 100, -(2.0 ** 127), 3.0, 0.0, 2.0 ** -120, -(2.0 ** -112), 0.0, 0.0, float("inf"), 1.5, -2.0, 0.0,
                        float("nan"), -3.0, float("-inf"), 7.0, -0.0, 0.0, 0.0, 0.0, 1.0, -(2.0 ** -20), 2.0 ** -30, 0.0, 255 / 128, -255 / 128])
    F, N = len(row), 70
    x = torch.zeros(N, 32, device="cuda", dtype=BF16)
    x[:, 0] = 1
    w = torch.zeros(F, 32, device="cuda", dtype=BF16)
    w[:, 0] = row.to(BF16)
    y, kept = torch.empty(N, F, device="cuda", dtype=BF16), torch.empty(N, (F + 3) // 4 * 4, device="cuda", dtype=BF16)
    assert L.tgt_linear_epilogue_fwd(x.data_ptr(), w.data_ptr(), None, None, N, 32, F, _lib.DTYPE_BF16, 2, y.data_ptr(), kept.data_ptr(), None, 0, st) == 0
    got, want = unpacked(kept)[:, :F], w[:, 0].double().cpu().repeat(N, 1)
    most = torch.nn.functional.pad(want, (0, -F % 4)).view(N, -1, 4)
    finite = torch.isfinite(most).all(2, keepdim=True).expand_as(most).flatten(1)[:, :F]
    bound = (2.0 ** -12 * most.abs().amax(2, keepdim=True).clamp(min=2.0 ** -114)).expand_as(most).flatten(1)[:, :F]
    assert ((got - want).abs() <= bound)[finite].all() and torch.equal(got[finite].sign(), want[finite].sign())
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[:, 12:19].nan_to_num(), want[:, 12:19].nan_to_num())
    assert L.tgt_linear_epilogue_fwd(x.data_ptr(), w.data_ptr(), None, None, N, 32, F, _lib.DTYPE_BF16, 2, y.data_ptr(), kept.data_ptr() + 2, None, 0, st) == _lib.ERR_INVALID_ARG


def test_kept_or_formed_again(cuda):
    """The C entry points take both ways at any size: kept values are the products, and the gradients of either way agree with the formula."""
    L = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    for dt, code in ((F32, 0), (BF16, 1)):
        for N, K, F in ((40, 64, 48), (200, 72, 96), (200, 72, 97), (130, 520, 1032)):
            x, wg, wu, bg, bu, dh = gated_case(N, K, F, dt, "silu", True)
            P = [t.data_ptr() for t in (x, wg, wu, bg, bu)]
            for keep in (False, True):
                kept, h = torch.empty(N, 2, F if dt == F32 else (F + 3) // 4 * 4, device="cuda", dtype=dt), torch.empty(N, F, device="cuda", dtype=dt)
                kp = kept.data_ptr() if keep else None
                nbytes = L.tgt_gated_linear_fwd_workspace_bytes(N, K, F, code)
                ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
                assert L.tgt_gated_linear_fwd(*P, N, K, F, code, 3, h.data_ptr(), kp, ws.data_ptr(), nbytes, st) == 0
                nbytes = L.tgt_gated_linear_bwd_workspace_bytes(N, K, F, code)
                ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
                outs = {"h": h, "x": torch.empty_like(x), "wg": torch.empty_like(wg), "wu": torch.empty_like(wu), "bg": torch.empty_like(bg), "bu": torch.empty_like(bu)}
                import ctypes
                dW = (ctypes.c_void_p * 2)(outs["wg"].data_ptr(), outs["wu"].data_ptr())
                db = (ctypes.c_void_p * 2)(outs["bg"].data_ptr(), outs["bu"].data_ptr())
                assert L.tgt_gated_linear_bwd(*P, dh.data_ptr(), N, K, F, code, 3, kp, outs["x"].data_ptr(), dW, db, ws.data_ptr(), nbytes, st) == 0
                check_gated(x, wg, wu, bg, bu, dh, "silu", outs, kept=keep)
                if keep:
                    for at, w, b in ((0, wg, bg), (1, wu, bu)):
                        m = Kept(Mapped(d(x), d(w), d(b)), dt)
                        near(kept[:, at] if dt == F32 else unpacked(kept[:, at])[:, :F], m.v, m.e, "kept")


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("act", ["relu", None])
def test_gated_linear_other_activations(cuda, dt, act):
    case = gated_case(100, 48, 72, dt, act, True)
    check_gated(*case, act, run_gated(*case, act))


# A stretch of the contraction for each half or quarter of a matrix instruction's rows, row blocks of 16 and 32, contractions and columns that end inside them
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 8, 9, 20, 40, 64])
@pytest.mark.parametrize("shape", [(4096, 70), (2056, 1030), (1023, 13), (5000, 2050)])
def test_few_rows_of_long_contractions(cuda, dt, rows, shape):
    K, F = shape
    x, wg, wu, bg, bu, _ = gated_case(rows, K, F, dt, "silu", True)
    with torch.no_grad():
        check_gated(x, wg, wu, bg, bu, None, "silu", {"h": T.gated_linear(x, wg, wu, bg, bu)})
        x, w, b, r, _ = linear_case(rows, K, F, dt, True, True)
        check_linear(x, w, b, r, None, "gelu", {"y": T.linear_act(x, w, b, "gelu", r)})


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 7, 15, 16, 17, 31, 32, 33, 64])
@pytest.mark.parametrize("shape", [(64, 96), (1024, 200), (2000, 33), (77, 130)])
def test_gated_linear_few_rows_without_gradients(cuda, dt, rows, shape):
    K, F = shape
    x, wg, wu, bg, bu, _ = gated_case(rows, K, F, dt, "silu", True)
    with torch.no_grad():
        check_gated(x, wg, wu, bg, bu, None, "silu", {"h": T.gated_linear(x, wg, wu, bg, bu)})


def test_gated_linear_gradient_is_that_of_differences(cuda):
    """float32 against central differences of the formula in 64 bits: what remains is the float32 arithmetic, 1e-5 of the largest gradient."""
    x, wg, wu, bg, bu, dh = gated_case(6, 12, 10, F32, "gelu", True)
    outs = run_gated(x, wg, wu, bg, bu, dh, "gelu")
    args = {k: d(v) for k, v in dict(x=x, wg=wg, wu=wu, bg=bg, bu=bu).items()}
    DH = d(dh)

    def f():
        return (act64("gelu", args["x"] @ args["wg"].T + args["bg"]) * (args["x"] @ args["wu"].T + args["bu"]) * DH).sum()

    for k, t in args.items():
        want, flat, step = torch.empty_like(t), t.view(-1), 1e-5
        for i in range(flat.numel()):
            keep = float(flat[i])
            flat[i] = keep + step
            up = f()
            flat[i] = keep - step
            want.view(-1)[i] = (up - f()) / (2 * step)
            flat[i] = keep
        near(outs[k], want, torch.full_like(want, 1e-5 * float(want.abs().max())), k)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows", [40, 400])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_activations_of_any_argument(cuda, act, dt, rows):
    """One feature, weight one: values and slopes over the whole range, kernels for few rows and for many.  float32: 2^-20 of 1 + |u|, what a few units in the last
    place of exp and a distribution function near one may cost; bfloat16 half a step more."""
    g = torch.Generator().manual_seed(2)
    big = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 20.0, -20.0, 60.0, -60.0, 88.0, -88.0, 104.0, -104.0, 1e4, -1e4, 1e30, -1e30])
    x = torch.cat([big, rand(g, rows - len(big), scale=3, device="cpu")]).to(dt).cuda()[:, None]
    one = torch.ones(1, 1, device="cuda", dtype=dt)
    xl = x.clone().requires_grad_(True)
    y = T.linear_act(xl, one, activation=act)
    (gx,) = torch.autograd.grad(y, xl, torch.ones_like(y))
    u = d(x)
    want = act64(act, u)
    near(y, want, half_step(dt) * want.abs() + fine(dt) * torch.minimum(1 + u.abs(), 1 + want.abs()), "value")
    s = slope64(act, u).nan_to_num(0)
    near(gx, s, 2 * half_step(dt) * s.abs() + fine(dt) * 4, "slope")
    with torch.no_grad():
        near(T.linear_act(x, one, activation=act), want, half_step(dt) * want.abs() + fine(dt) * torch.minimum(1 + u.abs(), 1 + want.abs()), "value")
        h = T.gated_linear(x, one, 0 * one, up_bias=one[0], activation=act)      # act(u) * 1
        near(h, want, half_step(dt) * want.abs() + fine(dt) * torch.minimum(1 + u.abs(), 1 + want.abs()), "gated")


def test_only_some_gradients_wanted(cuda):
    x, wg, wu, bg, bu, dh = gated_case(50, 32, 48, F32, "silu", True)
    full = run_gated(x, wg, wu, bg, bu, dh, "silu")
    for wanted in (("x",), ("wg",), ("wu", "bu"), ("bg",), ("x", "bu")):
        leaves = {k: v.detach().clone().requires_grad_(k in wanted) for k, v in dict(x=x, wg=wg, wu=wu, bg=bg, bu=bu).items()}
        h = T.gated_linear(*leaves.values())
        for k, got in zip(wanted, torch.autograd.grad(h, [leaves[k] for k in wanted], dh)):
            assert torch.equal(got, full[k]), (wanted, k)


# ---- linear with an epilogue -----------------------------------------------------------------------------------------------------------------

def linear_case(N, K, M, dt, bias, residual):
    g = torch.Generator().manual_seed(N * 5 + K * 11 + M)
    return (rand(g, N, K, dt=dt), rand(g, M, K, dt=dt, scale=1.2 / math.sqrt(K)), rand(g, M, dt=dt, scale=0.3) if bias else None,
            rand(g, N, M, dt=dt) if residual else None, rand(g, N, M, dt=dt))


def check_linear(x, w, b, r, dy, act, outs, eight=False, kept=False):
    dt = outs["y"].dtype
    X, W, B, R, DY = d(x), d(w), d(b), d(r), d(dy)
    u = Mapped(X, W, B, eight=eight)
    y, ey = act64(act, u.v), 1.13 * u.e + (fine(dt) * (u.v.abs() + u.e) if act else 0)
    if r is not None:
        y = y + R
        ey = ey + 2.0 ** -23 * (y.abs() + R.abs())
    near(outs["y"], y, stored(y, ey, dt), "y")
    if dy is None:
        return
    if act is None:
        du, edu = DY, torch.zeros_like(DY)
    else:
        if kept:
            u = Kept(u, dt)
        du = DY * slope64(act, u.v)
        edu = stored(du, DY.abs() * (curve(act, u.v, u.e, getattr(u, "edge", None)) + fine(dt) * (1 + u.v.abs())) + 2.0 ** -22 * du.abs(), dt)
    dx, dw = Mapped(du, W.T, ea=edu), Mapped(du.T, X.T, ea=edu.T)
    near(outs["x"], dx.v, stored(dx.v, dx.e, dt), "dx")
    near(outs["w"], dw.v, stored(dw.v, dw.e, dt), "dW")
    if b is not None:
        db, edb = du.sum(0), edu.sum(0) + sums(len(X)) * du.abs().sum(0)
        near(outs["b"], db, stored(db, edb, dt), "db")
    if r is not None:
        assert torch.equal(outs["r"], dy)


def run_linear(x, w, b, r, dy, act):
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in dict(x=x, w=w, b=b, r=r).items() if v is not None}
    y = T.linear_act(leaves["x"], leaves["w"], leaves.get("b"), activation=act, residual=leaves.get("r"))
    return {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act,bias,residual", [(None, True, True), ("gelu", True, False), ("silu", False, True)])
def test_linear_act(cuda, shape, dt, act, bias, residual):
    case = linear_case(*shape, dt, bias, residual)
    check_linear(*case, act, run_linear(*case, act))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 4, 16, 17, 33, 64])
@pytest.mark.parametrize("shape", [(64, 96), (4096, 128), (2000, 33), (77, 130)])
def test_linear_act_few_rows_without_gradients(cuda, dt, rows, shape):
    x, w, b, r, _ = linear_case(rows, *shape, dt, True, True)
    with torch.no_grad():
        check_linear(x, w, b, r, None, "relu", {"y": T.linear_act(x, w, b, "relu", r)})


# ---- norm --------------------------------------------------------------------------------------------------------------------------------------

WIDTHS = [1, 2, 3, 7, 8, 32, 40, 47, 64, 100, 128, 250, 256, 300, 512, 768, 1000, 1024, 1408, 2048, 2050, 4096, 5001, 8192, 12000, 16384]


def norm_case(N, C, dt, residual):
    g = torch.Generator().manual_seed(N * 31 + C)
    return rand(g, N, C, dt=dt), rand(g, N, C, dt=dt) if residual else None, (1 + rand(g, C, scale=0.2)).to(dt), rand(g, N, C, dt=dt), rand(g, N, C, dt=dt)


# of a row's mean: a thread adds up at most 64 values, threads are added in a tree of at most 10 levels and 16 waves in turn
MEAN = 100 * 2.0 ** -24


def check_norm(x, r, w, dy, ds, outs):
    dt = x.dtype
    s = d(x if r is None else (x.float() + r.float()).to(dt))
    assert torch.equal(d(outs["s"]), s)
    W = d(w)
    rstd = 1 / (s.square().mean(1, keepdim=True) + EPS).sqrt()
    xh = s * rstd
    y = xh * W
    near(outs["y"], y, stored(y, y.abs() * (MEAN + 2.0 ** -21), dt), "y")
    if dy is None:
        return
    DY, DS = d(dy), d(ds)
    g = DY * W
    m = (g * xh).mean(1, keepdim=True)
    grad = rstd * (g - xh * m) + DS
    e = (MEAN + 2.0 ** -20) * rstd * (g.abs() + xh.abs() * (m.abs() + (g * xh).abs().mean(1, keepdim=True))) + 2.0 ** -23 * (DS.abs() + grad.abs())
    near(outs["x"], grad, stored(grad, e, dt), "ds")
    if r is not None:
        assert torch.equal(outs["r"], outs["x"])
    dw = (DY * xh).sum(0)
    near(outs["w"], dw, stored(dw, (sums(len(s)) + MEAN + 2.0 ** -20) * (DY * xh).abs().sum(0), dt), "dw")


def run_norm(x, r, w, dy, ds):
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in dict(x=x, r=r, w=w).items() if v is not None}
    s, y = T.add_rms_norm(leaves["x"], leaves.get("r"), leaves["w"], EPS)
    return {"s": s, "y": y, **dict(zip(leaves, torch.autograd.grad((s, y), list(leaves.values()), (ds, dy))))}


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("C", WIDTHS)
def test_add_rms_norm(cuda, dt, C):
    for N, residual in ((1, True), (37, False), (700, True)):
        case = norm_case(N, C, dt, residual)
        check_norm(*case, run_norm(*case))
        with torch.no_grad():
            s, y = T.add_rms_norm(*case[:3], EPS)
            check_norm(*case[:3], None, None, {"s": s, "y": y})


def test_norm_gradient_without_one_of_the_outputs(cuda):
    x, r, w, dy, ds = norm_case(33, 96, F32, True)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    s, y = T.add_rms_norm(*leaves, EPS)
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    check_norm(x, r, w, dy, torch.zeros_like(ds), {"s": s, "y": y, **dict(zip("xrw", only_y))})
    only_s = torch.autograd.grad(s, leaves, ds, allow_unused=True)
    assert torch.equal(only_s[0], ds) and torch.equal(only_s[1], ds) and (only_s[2] is None or not only_s[2].any())


def check_codes(y, e, codes, scales):
    """codes and scales against y (64 bits, off by e at most)"""
    scales = d(scales)
    top = y.abs().amax(1)
    et = e.amax(1)
    assert torch.equal(torch.exp2(scales.log2().round()), scales)
    zero = top == 0
    assert (scales[zero] == 1).all()
    s, t, et = scales[~zero], top[~zero], et[~zero]
    assert (t - et <= 448 * s).all() and ((t + et > 224 * s) | (s == 2.0 ** -126)).all()
    near(codes.float().cpu().double() * scales[:, None], y, 2.0 ** -4 * y.abs() + scales[:, None] * 2.0 ** -10 + 1.07 * e, "codes")


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("C", [1, 5, 16, 64, 100, 256, 1000, 1408, 2048, 4096, 8192, 16384])
def test_add_rms_norm_8bit(cuda, dt, C):
    for N, residual in ((1, False), (65, True)):
        x, r, w, _, _ = norm_case(N, C, dt, residual)
        s, codes, scales = T.add_rms_norm_8bit(x, r, w, EPS)
        assert codes.dtype == E4M3 and codes.shape == x.shape and scales.shape == (N,)
        S = d(s)
        assert torch.equal(S, d(x if r is None else (x.float() + r.float()).to(dt)))
        y = S / (S.square().mean(1, keepdim=True) + EPS).sqrt() * d(w)
        check_codes(y, y.abs() * (MEAN + 2.0 ** -21), codes, scales)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_quantize_rows_is_exact(cuda, dt):
    g = torch.Generator().manual_seed(3)
    for N, C in ((1, 1), (7, 33), (64, 256), (9, 5000), (2, 16384)):
        w = rand(g, N, C, dt=dt) * torch.exp2(torch.randint(-60, 60, (N, 1), generator=g)).to(dt).cuda()
        if N > 2:
            w[1] = 0
            w[2, 0] = 1.7e38 if dt == F32 else 1e38
            w[3] = 1e-39 if dt == F32 else 2.0 ** -130
            w[4] = torch.where(torch.rand(C, generator=g).cuda() < 0.5, 448.0, -300.0).to(dt)
            w[5] = torch.where(torch.rand(C, generator=g).cuda() < 0.5, 450.0, 0.015625).to(dt)
        codes, scales = T.quantize_rows(w)
        W = d(w)
        check_codes(W, torch.zeros_like(W), codes, scales)
        want = (W / d(scales)[:, None]).float().to(E4M3)      # (a power of two: exact)
        assert torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))
    w = torch.tensor([[1.0, float("nan"), 2.0], [float("inf"), 1.0, -2.0]], device="cuda", dtype=dt)
    codes, _ = T.quantize_rows(w)
    assert codes.float().isnan().tolist() == [[False, True, False], [True, False, False]]


# ---- operands in 8 bits -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 16, 1), (1, 1024, 96), (7, 64, 33), (17, 48, 130), (130, 128, 64), (300, 272, 140), (64, 4096, 100), (3, 4096, 70), (7, 2064, 1030), (40, 4096, 70), (200, 4096, 130), (300, 1040, 520), (65, 2048, 264)])
def test_products_in_8_bits(cuda, out, shape):
    N, K, F = shape
    g = torch.Generator().manual_seed(K + F)
    x, xs = T.quantize_rows(rand(g, N, K) * 3)
    (wg, gs), (wu, us) = (T.quantize_rows(rand(g, F, K, scale=1.2 / math.sqrt(K))) for _ in range(2))
    bg, bu, r = rand(g, F, dt=out, scale=0.3), rand(g, F, dt=out, scale=0.3), rand(g, N, F, dt=out)

    def value(c, s):
        return c.float().double().cpu() * d(s)[:, None]

    X, WG, WU = value(x, xs), value(wg, gs), value(wu, us)
    for b1, b2, act in ((None, None, "silu"), (bg, bu, "gelu")):
        h = T.gated_linear_8bit(x, xs, wg, gs, wu, us, b1, b2, activation=act, dtype=out)
        assert h.dtype == out
        p, q = Mapped(X, WG, d(b1), eight=True), Mapped(X, WU, d(b2), eight=True)
        a = act64(act, p.v)
        ea = 1.13 * p.e + fine(out) * (p.v.abs() + p.e)
        want = a * q.v
        near(h, want, stored(want, ea * (q.v.abs() + q.e) + a.abs() * q.e + 2.0 ** -23 * want.abs(), out), "h")
    for b1, r1, act in ((None, None, None), (bg, r, "relu")):
        y = T.linear_act_8bit(x, xs, wg, gs, b1, act, r1, dtype=out)
        check_linear(X, WG, d(b1), d(r1), None, act, {"y": y}, eight=True)


# ---- how they are called ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", [F32, BF16])
def test_leading_dimensions_strides_and_addresses(cuda, dt):
    """Batches of rows, transposed and expanded tensors, slices that start at any element: the same bits as a compact copy gives at an aligned address, or
    bounds hold where another variant takes the call."""
    x, wg, wu, bg, bu, dh = gated_case(60, 40, 56, dt, "silu", True)
    want = run_gated(x, wg, wu, bg, bu, dh, "silu")

    def odd(t):      # the same values one element behind an aligned address
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    got = run_gated(x.view(3, 4, 5, 40), wg.T.contiguous().T, wu, bg, bu, dh.view(3, 4, 5, 56), "silu")
    assert got["h"].shape == (3, 4, 5, 56) and got["x"].shape == (3, 4, 5, 40)
    for k in want:
        assert torch.equal(got[k].reshape(want[k].shape), want[k]), k
    leaves = [odd(t).detach().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    h = T.gated_linear(*leaves)
    check_gated(x, wg, wu, bg, bu, dh, "silu", {"h": h, **dict(zip(("x", "wg", "wu", "bg", "bu"), torch.autograd.grad(h, leaves, odd(dh))))})
    (gx,) = torch.autograd.grad(T.gated_linear(leaves[0], *leaves[1:]).sum(), leaves[:1])      # an expanded gradient
    ones = run_gated(x, wg, wu, bg, bu, torch.ones_like(dh), "silu")
    near(gx, d(ones["x"]), 0.05 * d(ones["x"]).abs() + 0.05, "dx of a sum")

    lx, lw, lb, lr, ldy = linear_case(60, 40, 56, dt, True, True)
    leaves = [odd(t).detach().requires_grad_(True) for t in (lx, lw, lb, lr)]
    y = T.linear_act(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
    check_linear(lx, lw, lb, lr, ldy, "gelu", {"y": y, **dict(zip(("x", "w", "b", "r"), torch.autograd.grad(y, leaves, odd(ldy))))})

    nx, nr, nw, ndy, nds = norm_case(60, 40, dt, True)
    leaves = [odd(t).detach().requires_grad_(True) for t in (nx, nr, nw)]
    s, y = T.add_rms_norm(*leaves, EPS)
    check_norm(nx, nr, nw, ndy, nds, {"s": s, "y": y, **dict(zip("xrw", torch.autograd.grad((s, y), leaves, (odd(nds), odd(ndy)))))})
    c1, c2 = T.add_rms_norm_8bit(odd(nx), odd(nr), odd(nw), EPS), T.add_rms_norm_8bit(nx.T.contiguous().T, nr, nw, EPS)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(c1, c2))


@pytest.mark.parametrize("dt", [F32, BF16])
def test_no_rows(cuda, dt):
    x, wg, wu, bg, bu, dh = gated_case(4, 24, 32, dt, "silu", True)
    got = run_gated(x[:0], wg, wu, bg, bu, dh[:0], "silu")
    assert got["h"].shape == (0, 32) and got["x"].shape == (0, 24)
    assert all(not got[k].any() for k in ("wg", "wu", "bg", "bu"))
    got = run_linear(x[:0], wg, bg, None, dh[:0], "gelu")
    assert got["y"].shape == (0, 32) and not got["w"].any() and not got["b"].any()
    nx, nr, nw, ndy, nds = norm_case(3, 24, dt, True)
    got = run_norm(nx[:0], nr[:0], nw, ndy[:0], nds[:0])
    assert got["y"].shape == (0, 24) and not got["w"].any()
    s, codes, scales = T.add_rms_norm_8bit(nx[:0], None, nw)
    assert codes.shape == (0, 24) and scales.shape == (0,)
    assert T.linear_act_8bit(*T.quantize_rows(torch.zeros(0, 16, device="cuda")), *T.quantize_rows(torch.ones(3, 16, device="cuda"))).shape == (0, 3)


def test_same_inputs_same_bits(cuda):
    """Also where weight gradients are cut along the nodes."""
    for dt in (F32, BF16):
        case = gated_case(5000, 64, 80, dt, "silu", True)
        a, b = run_gated(*case, "silu"), run_gated(*case, "silu")
        assert all(torch.equal(a[k], b[k]) for k in a)
        check_gated(*case, "silu", a)
        case = norm_case(3000, 64, dt, True)
        a, b = run_norm(*case), run_norm(*case)
        assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("rows", [3, 200])
def test_infinities_and_nans_stay_in_their_rows(cuda, rows):
    """An infinity in x or W gives the infinities that multiply-adds give (float32 goes through three parts, one of them zero), a NaN a NaN in its row
    only; the largest numbers do not overflow on their way."""
    for dt in (F32, BF16):
        x = torch.ones(rows, 96, device="cuda", dtype=dt)
        w = torch.full((40, 96), 0.5, device="cuda", dtype=dt)
        x[0, 5], x[1, 7], w[3, 9] = float("inf"), float("nan"), float("-inf")
        x[2, 11] = torch.finfo(dt).max
        y = T.linear_act(x, w).double()
        want = x.double().cpu() @ w.double().cpu().T
        assert torch.equal(y.isnan().cpu(), want.isnan())
        assert torch.equal(y.isinf().cpu(), want.isinf())
        ok = want.isfinite()
        near(y.cpu()[ok], want[ok], want[ok].abs() * (half_step(dt) + sums(96)), "finite ones")
        xl = x.clone().requires_grad_(True)
        wl = w.clone().requires_grad_(True)
        dy = torch.ones(rows, 40, device="cuda", dtype=dt)
        gx, gw = torch.autograd.grad(T.linear_act(xl, wl), (xl, wl), dy)
        assert torch.equal(gx.isinf().cpu(), (torch.ones(rows, 40).double() @ w.double().cpu()).isinf())
        wantw = torch.ones(40, rows).double() @ x.double().cpu()
        assert torch.equal(gw.isinf().cpu(), wantw.isinf()) and torch.equal(gw.isnan().cpu(), wantw.isnan())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_infinities_in_contractions_in_pieces(cuda, dt):
    """The same where a contraction is cut in pieces: infinities in several pieces, of both weights of the input gradient."""
    N, K, F = 300, 2048, 1032
    x, w = torch.ones(N, K, device="cuda", dtype=dt), torch.full((F, K), 0.5, device="cuda", dtype=dt)
    x[0, 5], x[1, 2000], x[2, 700], x[2, 1900], w[3, 1500], w[4, 9], w[4, 1999] = float("inf"), float("nan"), float("inf"), float("-inf"), float("-inf"), float("inf"), float("inf")
    y, want = T.linear_act(x, w).double().cpu(), x.double().cpu() @ w.double().cpu().T
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf()) and torch.equal(y[want.isfinite()], want[want.isfinite()])
    N, K, F = 70, 264, 2048
    x, wg = torch.full((N, K), 0.25, device="cuda", dtype=dt), torch.full((F, K), 0.125, device="cuda", dtype=dt)
    dh = torch.ones(N, F, device="cuda", dtype=dt)
    for at in ((), (5,), (2000,), (5, 2000), (1023, 1024)):
        for which in (0, 1):
            W = [wg.clone(), wg.clone()]
            for k, f in enumerate(at):
                dh[3] = 0
                dh[4, f] = float("inf")
                W[which][f, 7 + k] = float("inf")
            xl, gl, ul = (t.clone().requires_grad_(True) for t in (x, *W))
            dx = torch.autograd.grad(T.gated_linear(xl, gl, ul, activation="relu"), xl, dh)[0].double().cpu()
            X, WG, WU, DH = d(x), d(W[0]), d(W[1]), d(dh)
            g, u = X @ WG.T, X @ WU.T
            want = (DH * u * (g > 0)) @ WG + (DH * g.clamp(min=0)) @ WU
            assert torch.equal(dx.isnan(), want.isnan()) and torch.equal(dx.isinf(), want.isinf()), (at, which)
            assert (dx - want).abs()[want.isfinite()].le(want.abs()[want.isfinite()] * (3 * half_step(dt) + sums(2 * F + K) * 3)).all()


def test_norm_of_a_row_with_a_nan_and_of_zeros(cuda):
    for dt in (F32, BF16):
        x = torch.ones(5, 100, device="cuda", dtype=dt)
        x[1, 3] = float("nan")
        x[2] = 0
        w = torch.ones(100, device="cuda", dtype=dt)
        _, y = T.add_rms_norm(x, None, w)
        assert y[1].isnan().all() and y[[0, 2, 3, 4]].isfinite().all() and not y[2].any()
        _, codes, scales = T.add_rms_norm_8bit(x, None, w)
        assert codes[1].float().isnan().all() and scales[2] == 1 and not codes[2].float().any()


@pytest.mark.parametrize("shape", [(300, 64, 96), (300, 2048, 264)])
def test_on_another_stream(cuda, shape):
    """And on two streams at once: neither call's workspaces are the other's."""
    case = gated_case(*shape, BF16, "silu", True)
    want = run_gated(*case, "silu")
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for side in sides:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(run_gated(*case, "silu"))
    for side in sides:
        side.synchronize()
    assert all(torch.equal(o[k], want[k]) for o in got for k in want)


def chain(x, r, wn, wg, wu, wd, b):
    s, y = T.add_rms_norm(x, r, wn)
    return T.linear_act(T.gated_linear(y, wg, wu), wd, b, residual=s)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("sizes", [(200, 64, 160), (300, 1032, 528), (40, 2048, 200)])
def test_a_block_captured_and_replayed(cuda, dt, sizes):
    """Norm, gated projections, projection back with the residual: forward and backward in a graph, replayed on new inputs with other work between."""
    g = torch.Generator().manual_seed(5)
    N, C, F = sizes
    params = [(1 + rand(g, C, scale=0.1)).to(dt), rand(g, F, C, dt=dt, scale=0.15), rand(g, F, C, dt=dt, scale=0.15), rand(g, C, F, dt=dt, scale=0.1), rand(g, C, dt=dt)]
    x, r, dy = (rand(g, N, C, dt=dt) for _ in range(3))

    def step(x, r, dy):
        leaves = [t.detach().requires_grad_(True) for t in [x, r] + params]
        y = chain(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, r, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, r, dy)
    for i in range(4):
        for t in (x, r, dy):
            t.copy_(rand(g, *t.shape, dt=dt))
        want = step(x, r, dy)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_a_block_in_8_bits(cuda):
    """As a serving program calls them: weights in 8 bits once, then norm -> gated projections in 8 bits -> projection back in bfloat16, for one row and for
    many, against the same in 64 bits on the codes."""
    g = torch.Generator().manual_seed(9)
    C, F = 128, 272
    wn = (1 + rand(g, C, scale=0.1)).to(BF16)
    (wg, gs), (wu, us) = (T.quantize_rows(rand(g, F, C, dt=BF16, scale=0.1)) for _ in range(2))
    wd = rand(g, C, F, dt=BF16, scale=0.1)
    for N in (1, 5, 140):
        x, r = rand(g, N, C, dt=BF16), rand(g, N, C, dt=BF16)
        s, codes, scales = T.add_rms_norm_8bit(x, r, wn)
        h = T.gated_linear_8bit(codes, scales, wg, gs, wu, us)
        y = T.linear_act(h, wd, residual=s)
        X = codes.float().double().cpu() * d(scales)[:, None]
        p, q = (Mapped(X, c.float().double().cpu() * d(sc)[:, None], eight=True) for c, sc in ((wg, gs), (wu, us)))
        want = act64("silu", p.v) * q.v
        near(h, want, stored(want, (1.13 * p.e + fine(BF16) * p.v.abs()) * (q.v.abs() + q.e) + p.v.abs() * q.e, BF16), "h")
        check_linear(h, wd, None, s, None, None, {"y": y})
        # one row of many is what it is alone, to the order of its sums
        s1, c1, sc1 = T.add_rms_norm_8bit(x[:1], r[:1], wn)
        assert torch.equal(c1.float(), codes[:1].float()) and torch.equal(sc1, scales[:1])


def test_gated_graphormer_learns_its_gradients(cuda):
    """Graphormer(gated=True): one step against the same modules written out with torch, float32."""
    from torchgt_amd import workloads
    e, n = workloads.barabasi_albert(n=200, m=3, seed=1)
    ei = torch.from_numpy(e).cuda()
    torch.manual_seed(0)
    m = T.Graphormer(2, 4, 16, 32, 7, 1, 0.0, 0.0, 0.0, 64, 1, gated=True).cuda()
    for p in m.parameters():
        p.data.add_(torch.randn_like(p) * 0.1)
    N = n - 1
    x = torch.randn(N, 16, device="cuda")
    y = m(x, None, ei, attn_type="sparse")
    assert y.shape == (N, 7)
    target = torch.randint(0, 7, (N,), device="cuda")
    T.nll_loss(y, target).backward()

    from torch.func import functional_call  # noqa: F401
    params = {k: v.detach().double().cpu().requires_grad_(True) for k, v in m.named_parameters()}

    def lin(t, name):
        return t @ params[name + ".weight"].T + params[name + ".bias"]

    def rms(t, name):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * params[name + ".weight"]

    from oracle import sparse_attention as osa
    h = torch.cat([params["graph_token.weight"], lin(d(x), "node_encoder")])
    for i in range(2):
        at = f"layers.{i}."
        z = rms(h, at + "self_attention_norm")
        q, k, v = (lin(z, at + f"self_attention.linear_{c}").view(-1, 4, 8) for c in "qkv")
        a = osa.sparse_attention(q, k, v, ei.cpu(), None)[0].reshape(-1, 32)
        h = h + lin(a, at + "self_attention.output_layer")
        z = rms(h, at + "ffn_norm")
        h = h + lin(act64("silu", lin(z, at + "ffn.gate")) * lin(z, at + "ffn.up"), at + "ffn.down")
    want = torch.log_softmax(lin(rms(h, "final_ln")[1:], "downstream_out_proj"), 1)
    # the framework's float32 bound on outputs and gradients of whole models: 1e-4 of the largest value
    near(y, want.detach(), torch.full_like(want, 1e-4 * float(want.detach().abs().max())), "log probabilities")
    torch.nn.functional.nll_loss(want, target.cpu()).backward()
    for k, p in m.named_parameters():
        if params[k].grad is None:
            assert p.grad is None, k
            continue
        near(p.grad, params[k].grad, torch.full_like(params[k].grad, 1e-4 * float(params[k].grad.abs().max()) + 1e-7), k)
    # with dropout at work the block's residual waits for the next norm: rate 0 in training against eval, then a rate that drops
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(x, None, ei, attn_type="sparse"), y.detach())
    m.train()
    for layer in m.layers:
        layer.ffn_dropout.p = 0.5
    assert m(x, None, ei, attn_type="sparse").isfinite().all()


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------------------

def test_refusals(cuda):
    x, wg, wu, bg, bu, dh = gated_case(8, 32, 48, F32, "silu", True)
    for bad in [lambda: T.gated_linear(x, wg.bfloat16(), wu), lambda: T.gated_linear(x, wg[:, :16], wu), lambda: T.gated_linear(x, wg, wu[:40]),
                lambda: T.gated_linear(x, wg, wu, bg[:5]), lambda: T.gated_linear(x.half(), wg.half(), wu.half()), lambda: T.gated_linear(x.cpu(), wg, wu),
                lambda: T.gated_linear(x, wg.cpu(), wu), lambda: T.gated_linear(x, wg, wu, bg.cpu()), lambda: T.linear_act(x, wg, residual=dh[:4]),
                lambda: T.linear_act(x, wg, residual=dh.bfloat16()), lambda: T.linear_act(x, wg, residual=dh.view(2, 4, 48)),
                lambda: T.linear_act(x, wg.view(-1)), lambda: T.add_rms_norm(x, None, wg[0][:5]), lambda: T.add_rms_norm(x, x[:4], wg[0]),
                lambda: T.add_rms_norm(x, x.bfloat16(), wg[0]), lambda: T.add_rms_norm(torch.zeros(2, 16385, device="cuda"), None, torch.zeros(16385, device="cuda")),
                lambda: T.quantize_rows(x.double()), lambda: T.add_rms_norm(torch.zeros(3, 0, device="cuda"), None, torch.zeros(0, device="cuda"))]:
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    with pytest.raises(ValueError, match="activation"):
        T.gated_linear(x, wg, wu, activation="tanh")
    c, s = T.quantize_rows(x)
    w, ws = T.quantize_rows(wg)
    for bad in [lambda: T.linear_act_8bit(x, s, w, ws), lambda: T.linear_act_8bit(c, s.double(), w, ws), lambda: T.linear_act_8bit(c, s[:3], w, ws),
                lambda: T.linear_act_8bit(c, s, w, ws, dtype=torch.float16), lambda: T.linear_act_8bit(c, s, w, ws, bg),
                lambda: T.linear_act_8bit(*T.quantize_rows(torch.ones(2, 24, device="cuda")), *T.quantize_rows(torch.ones(3, 24, device="cuda")))]:
        with pytest.raises(RuntimeError):
            bad()
    # no gradients in 8 bits, no second ones anywhere, no tangents
    with pytest.raises(RuntimeError, match="no gradient"):
        T.add_rms_norm_8bit(x.clone().requires_grad_(True), None, wg[0].contiguous())
    with pytest.raises(RuntimeError, match="no gradient"):
        T.quantize_rows(x.clone().requires_grad_(True))
    xl = x.clone().requires_grad_(True)
    for y in (T.gated_linear(xl, wg, wu), T.linear_act(xl, wg), T.add_rms_norm(xl, None, wg[0].contiguous())[1]):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(y.sum(), xl, create_graph=True)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            T.gated_linear(dual, wg, wu)


# ---- sizes that go to other variants -----------------------------------------------------------------------------------------------------------------

def sampled(rows, cols, g):
    return torch.randint(rows, (40,), generator=g), torch.randint(cols, (40,), generator=g)


@pytest.mark.parametrize("shape", [(16384, 256, 2048), (13000, 320, 2176), (12929, 328, 2184), (5000, 1288, 1480), (3001, 2048, 4352)])
def test_large_products_in_bf16(cuda, shape):
    """Whole tiles of 256 and what is left of them, against a float32 product of the same operands on the GPU (exact products, sums off by sums(n) of the magnitudes
    on either side), and element by element in 64 bits at sampled places with the last rows and columns among them."""
    N, K, F = shape
    x, wg, wu, bg, bu, dh = gated_case(N, K, F, BF16, "silu", True)
    outs = run_gated(x, wg, wu, bg, bu, dh, "silu")
    y = run_linear(x, wg, bg, dh, dh, "gelu")
    yn = run_linear(x, wg, bg, dh, dh, None)
    g = torch.Generator().manual_seed(1)
    rows = torch.cat([torch.tensor([0, N - 1, N - 2, (N - 1) // 256 * 256]), torch.randint(N, (28,), generator=g)])
    X, DH = d(x[rows]), d(dh[rows])
    check_gated(x[rows], wg, wu, bg, bu, None, "silu", {"h": outs["h"][rows]})
    check_linear(x[rows], wg, bg, dh[rows], None, "gelu", {"y": y["y"][rows]})
    check_linear(x[rows], wg, bg, dh[rows], None, None, {"y": yn["y"][rows]})
    WG, WU, BG, BU = d(wg), d(wu), d(bg), d(bu)

    def products(X, f=None):
        four = torch.arange(F) if f is None else (f[:, None] // 4 * 4 + torch.arange(4)).flatten()      # (F is a multiple of four)
        p, q = Mapped(X, WG[four], BG[four]), Mapped(X, WU[four], BU[four])
        if K >= 512:
            p, q = Kept(p, BF16), Kept(q, BF16)
        if f is not None:
            for m in (p, q):
                m.v, m.e = (t[:, torch.arange(len(f)) * 4 + f % 4] for t in (m.v, m.e))
        return p, q

    p, q = products(X)
    s, a = slope64("silu", p.v), act64("silu", p.v)
    dg, du = DH * q.v * s, DH * a
    edg = stored(dg, DH.abs() * (q.v.abs() * (0.8 * p.e + fine(BF16) * (1 + p.v.abs())) + (s.abs() + 0.8 * p.e) * q.e) + 2.0 ** -22 * dg.abs(), BF16)
    edu = stored(du, DH.abs() * (1.13 * p.e + fine(BF16) * (p.v.abs() + p.e)) + 2.0 ** -22 * du.abs(), BF16)
    dx = Mapped(torch.cat([dg, du], 1), torch.cat([WG, WU]).T, ea=torch.cat([edg, edu], 1))
    near(outs["x"][rows], dx.v, stored(dx.v, dx.e, BF16), "dx")
    dxn = Mapped(DH, WG.T)
    near(yn["x"][rows], dxn.v, stored(dxn.v, dxn.e, BF16), "dx of the linear")
    # weight gradients: sampled rows f, the last among them
    fs = torch.cat([torch.tensor([0, F - 1, F - 2, (F - 1) // 256 * 256]), torch.randint(F, (12,), generator=g)])
    X, DH = d(x), d(dh[:, fs])
    p, q = products(X, fs)
    s, a = slope64("silu", p.v), act64("silu", p.v)
    dg, du = DH * q.v * s, DH * a
    edg = stored(dg, DH.abs() * (q.v.abs() * (0.8 * p.e + fine(BF16) * (1 + p.v.abs())) + (s.abs() + 0.8 * p.e) * q.e) + 2.0 ** -22 * dg.abs(), BF16)
    edu = stored(du, DH.abs() * (1.13 * p.e + fine(BF16) * (p.v.abs() + p.e)) + 2.0 ** -22 * du.abs(), BF16)
    for got, v, e in ((outs["wg"], dg, edg), (outs["wu"], du, edu), (yn["w"], DH, torch.zeros_like(DH))):
        dw = Mapped(v.T, X.T, ea=e.T)
        near(got[fs], dw.v, stored(dw.v, dw.e, BF16), "dW")
    for got, v, e in ((outs["bg"], dg, edg), (outs["bu"], du, edu), (yn["b"], DH, torch.zeros_like(DH))):
        near(got[fs], v.sum(0), stored(v.sum(0), e.sum(0) + sums(N) * v.abs().sum(0), BF16), "db")
    again = run_gated(x, wg, wu, bg, bu, dh, "silu")
    assert all(torch.equal(outs[k], again[k]) for k in outs)


@pytest.mark.parametrize("shape", [(8200, 256, 2048), (5001, 1040, 2100), (2050, 2048, 6144)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_large_products_in_8_bits(cuda, shape, out):
    N, K, F = shape
    g = torch.Generator().manual_seed(K)
    x, xs = T.quantize_rows(rand(g, N, K, dt=BF16) * 3)
    (wg, gs), (wu, us) = (T.quantize_rows(rand(g, F, K, dt=BF16, scale=1.2 / math.sqrt(K))) for _ in range(2))
    bg, r = rand(g, F, dt=out, scale=0.3), rand(g, N, F, dt=out)
    h = T.gated_linear_8bit(x, xs, wg, gs, wu, us, bg, bg, dtype=out)
    y = T.linear_act_8bit(x, xs, wg, gs, bg, "relu", r, dtype=out)
    rows = torch.tensor([0, 1, 255, 256, N // 2, N - 2, N - 1])
    X = x[rows.cuda()].float().double().cpu() * d(xs[rows])[:, None]
    WG, WU = (c.float().double().cpu() * d(s)[:, None] for c, s in ((wg, gs), (wu, us)))
    p, q = Mapped(X, WG, d(bg), eight=True), Mapped(X, WU, d(bg), eight=True)
    a = act64("silu", p.v)
    want = a * q.v
    near(h[rows], want, stored(want, (1.13 * p.e + fine(out) * (p.v.abs() + p.e)) * (q.v.abs() + q.e) + a.abs() * q.e + 2.0 ** -23 * want.abs(), out), "h")
    check_linear(X, WG, d(bg), d(r[rows]), None, "relu", {"y": y[rows]}, eight=True)
