"""GPU: the row operators against plain 64-bit implementations, forward and backward.

Bounds are derived, not fitted.  u = 2^-24 is half a step of f32, s = finfo(dtype).eps / 2 half a step of the storage type.
A sum of n products accumulated in f32 in any order is off by at most about n u sum|terms|; every stored value by s of itself.
In bf16 the backward pass keeps the pre-activation as a half (2^-11) and rounds dz = dy act'(z) once: both appear as per-term errors.
"""
import math

import pytest
import torch
import torch.nn as nn

from srmi import autograd as AG
from srmi import rows
from test_rows_cpu import f32_product_rms

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TINY = 2.0 ** -120
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = {"none": None, "relu": nn.ReLU(), "lrelu": nn.LeakyReLU(0.2), "tanh": nn.Tanh(), "sigmoid": nn.Sigmoid(), "gelu": nn.GELU(),
        "gelu_tanh": nn.GELU(approximate="tanh"), "silu": nn.SiLU()}
# largest |act'| and |act''| (0 away from the kink of the piecewise linear ones)
LIP = {"none": 1, "relu": 1, "lrelu": 1, "tanh": 1, "sigmoid": 0.25, "gelu": 1.13, "gelu_tanh": 1.13, "silu": 1.1}
CURV = {"none": 0, "relu": 0, "lrelu": 0, "tanh": 0.77, "sigmoid": 0.097, "gelu": 0.8, "gelu_tanh": 0.8, "silu": 0.5}
# own error of the act / slope evaluation relative to max(|value|, |z|-scaled terms): bf16 uses the hardware's 2^x and reciprocal
FN = {"f32": 64 * U, "bf16": 2.0 ** -14}


def half_step(dt):
    return torch.finfo(DT[dt]).eps / 2


def act64(z, name):
    if name == "none":
        return z, torch.ones_like(z)
    zz = z.clone().requires_grad_()
    y = ACTS[name](zz) if name not in ("relu", "lrelu") else torch.where(zz > 0, zz, zz * (0.2 if name == "lrelu" else 0.0))
    (g,) = torch.autograd.grad(y.sum(), zz)
    return y.detach(), g


def assert_within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    excess = (got - want).abs() - bound
    k = int(excess.argmax())
    assert torch.isfinite(got).all() and float(excess.max()) <= 0, \
        f"{what}: |{float(got.flatten()[k])} - {float(want.flatten()[k])}| over its bound {float(bound.flatten()[k]):.3g}"


def make(shape, dt, gen, scale=1.0, pitch=0):
    wide = list(shape)
    if pitch:
        wide[-1] += pitch
    t = (torch.randn(wide, generator=gen) * scale).to(DT[dt]).to(DEV)
    return t[..., pitch:] if pitch else t


def linear_case(M, K, N, dt, act, bias, res, pitch, seed, lead=None):
    gen = torch.Generator().manual_seed(seed)
    x = make((lead or (M,)) + (K,) if not isinstance(lead, tuple) else lead + (K,), dt, gen, pitch=pitch)
    w = make((N, K), dt, gen, 1 / math.sqrt(max(K, 1)), pitch=pitch)
    b = make((N,), dt, gen, 0.1) if bias else None
    r = make(tuple(x.shape[:-1]) + (N,), dt, gen, pitch=pitch) if res else None
    dy = make(tuple(x.shape[:-1]) + (N,), dt, gen, pitch=pitch)
    leaves = [t.requires_grad_() if t is not None else None for t in (x, w, b, r)]
    return leaves, dy


def check_linear(leaves, dy, dt, act, run=None):
    x, w, b, r = leaves
    N, K = w.shape
    M = math.prod(x.shape[:-1])
    y = (run or (lambda: rows.linear(x, w, b, act=ACTS[act], residual=r)))()
    assert y.dtype == DT[dt] and y.is_contiguous() and y.shape == x.shape[:-1] + (N,)
    wanted = [t for t in leaves if t is not None]
    grads = dict(zip([k for k, t in zip("xwbr", leaves) if t is not None], torch.autograd.grad(y, wanted, dy)))

    x64, w64 = x.detach().double().cpu().reshape(M, K), w.detach().double().cpu()
    b64 = b.detach().double().cpu() if b is not None else torch.zeros(N, dtype=torch.float64)
    dy64 = dy.double().cpu().reshape(M, N)
    z = x64 @ w64.t() + b64
    f, g = act64(z, act)
    s, fn = half_step(dt), FN[dt]
    # z: K products + bias; the f32 path splits operands into three bf16 parts and drops products below 2^-24 (4 u)
    ez = (K + 8) * U * (x64.abs() @ w64.abs().t() + b64.abs())
    out = f + (r.detach().double().cpu().reshape(M, N) if r is not None else 0)
    ey = LIP[act] * ez + fn * (f.abs() + 0.01 * z.abs()) + 2 * U * out.abs() + s * out.abs() + TINY
    assert_within(y.reshape(M, N), out, ey + s * ey, f"y {act}")

    dz = dy64 * g
    zq = (2.0 ** -11 * z.abs() + 2.0 ** -25 if dt == "bf16" else 0) + ez                      # the kept pre-activation
    edz = dy64.abs() * (CURV[act] * zq + fn * (g.abs() + 0.01) * (act != "none"))
    if act in ("relu", "lrelu"):
        edz = edz + dy64.abs() * (z.abs() <= ez)                        # either slope within a rounding of the kink
    edz_q = edz + (s if act != "none" else 0) * (dz.abs() + edz)        # dz as the products read it (act none: dy itself)
    if "b" in grads:
        e = edz.sum(0) + (M + 8) * U * dz.abs().sum(0)
        want = dz.sum(0)
        assert_within(grads["b"], want, e * (1 + s) + s * want.abs() + TINY, f"db {act}")
    want = dz @ w64
    e = edz_q @ w64.abs() + (N + 8) * U * ((dz.abs() + edz_q) @ w64.abs())
    assert_within(grads["x"].reshape(M, K), want, e * (1 + s) + s * want.abs() + TINY, f"dx {act}")
    want = dz.t() @ x64
    e = edz_q.t() @ x64.abs() + (M + 8) * U * ((dz.abs() + edz_q).t() @ x64.abs())
    assert_within(grads["w"], want, e * (1 + s) + s * want.abs() + TINY, f"dw {act}")
    if r is not None:
        assert torch.equal(grads["r"], dy)


SIZES = [(1, 1, 1), (1, 16, 1), (2, 3, 5), (1, 1024, 264), (7, 64, 64), (16, 520, 72), (17, 1030, 33), (33, 2048, 16), (64, 96, 130),
         (65, 64, 256), (129, 257, 129), (256, 128, 256), (300, 512, 200), (1000, 40, 24), (515, 1152, 384),
         # fewer than eight columns on one side; K and M beyond 2048 (the longer k loop, sums split over workgroups); around 128 rows
         (200, 5, 70), (200, 70, 3), (130, 1, 1), (300, 2056, 200), (2500, 72, 40), (128, 33, 77), (127, 64, 64), (70, 4100, 90)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_sizes(M, K, N, dt):
    leaves, dy = linear_case(M, K, N, dt, "gelu", True, True, 0, 1000 * M + K + N)
    check_linear(leaves, dy, dt, "gelu")


# both sides of 16, 32 and 64 rows, short and long K, whole and ragged chunks of K (K % 8 != 0: rows off the 16-byte boundaries)
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("M", [1, 15, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("K,N", [(2048, 72), (2047, 33), (4104, 72), (4101, 35)])
def test_linear_few_rows(M, K, N, dt):
    leaves, dy = linear_case(M, K, N, dt, "lrelu", True, M % 2 == 0, 0, 10 * M + K)
    check_linear(leaves, dy, dt, "lrelu")


def _large(M, K, N, dt, seed):
    """y, dx, dw and db of act none against 64-bit products on the GPU; same bounds as check_linear"""
    leaves, dy = linear_case(M, K, N, dt, "none", True, False, 0, seed)
    x, w, b, _ = leaves
    y = rows.linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x64, w64, b64, dy64 = (t.detach().double() for t in (x, w, b, dy))
    s = half_step(dt)
    wt = w64.t().contiguous()
    dyt = dy64.t().contiguous()
    for got, want, mag, n in ((y, x64 @ wt + b64, x64.abs() @ wt.abs() + b64.abs(), K), (dx, dy64 @ w64, dy64.abs() @ w64.abs(), N),
                              (dw, dyt @ x64, dyt.abs() @ x64.abs(), M), (db, dy64.sum(0), dy64.abs().sum(0), M)):
        bound = (n + 8) * U * mag * (1 + s) + s * want.abs() + TINY
        assert float(((got.double() - want).abs() - bound).max()) <= 0


# enough tiles for each tile size, none of them whole: 256 x 256 in every product; f32 tiles of 128 with and without split sums
@pytest.mark.parametrize("M,K,N,dt", [(3590, 520, 3608, "bf16"), (3590, 3608, 520, "bf16"), (616, 3608, 3592, "bf16"), (1100, 2100, 1090, "f32"),
                                      (24000, 264, 136, "f32"), (2900, 300, 2950, "f32"), (1100, 2101, 1090, "bf16"), (24001, 263, 135, "bf16"),
                                      (40000, 64, 64, "bf16"), (40000, 64, 64, "f32")])
def test_linear_large(M, K, N, dt):
    _large(M, K, N, dt, M + K + N)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("bias,res", [(True, False), (False, True)])
def test_linear_activations(act, bias, res, dt):
    leaves, dy = linear_case(70, 96, 136, dt, act, bias, res, 0, 5)
    check_linear(leaves, dy, dt, act)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("pitch", [1, 8, 13])
def test_linear_strided_rows(pitch, dt):
    for M, K, N in ((5, 72, 40), (200, 136, 144)):
        leaves, dy = linear_case(M, K, N, dt, "silu", True, True, pitch, 6)
        check_linear(leaves, dy, dt, "silu")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("lead", [(), (3, 1, 5), (2, 7)])
def test_linear_leading_axes(lead, dt):
    leaves, dy = linear_case(None, 48, 24, dt, "none", True, False, 0, 7, lead=lead)
    check_linear(leaves, dy, dt, "none")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", [(0, 8, 5), (4, 0, 6), (4, 8, 0), (0, 0, 0), (300, 0, 40), (300, 8, 0)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_empty(M, K, N, dt, act):
    leaves, dy = linear_case(M, K, N, dt, act, True, True, 0, 8)
    check_linear(leaves, dy, dt, act)


def test_linear_transposed_and_broadcast_operands_are_copied():
    gen = torch.Generator().manual_seed(9)
    x = make((40, 9), "f32", gen).t().requires_grad_()                       # [9, 40], last axis strided
    w = make((40, 6), "f32", gen).t().requires_grad_()
    b = make((1,), "f32", gen).expand(6)
    y = rows.linear(x, w, b)
    torch.testing.assert_close(y, x @ w.t() + b, rtol=1e-5, atol=1e-5)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))                            # dy is an expanded scalar
    torch.testing.assert_close(gx, torch.ones_like(y) @ w, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(gw, torch.ones_like(y).t() @ x, rtol=1e-5, atol=1e-5)


def test_linear_broadcast_bias_gradient():
    gen = torch.Generator().manual_seed(10)
    x, w = make((50, 16), "f32", gen), make((6, 16), "f32", gen)
    b = make((1,), "f32", gen).requires_grad_()
    y = rows.linear(x, w, b.expand(6), act=nn.Tanh())
    (g,) = torch.autograd.grad(y, b, torch.ones_like(y))
    want = (1 - torch.tanh(x.double() @ w.double().t() + b.double()) ** 2).sum()
    assert abs(float(g) - float(want)) <= 300 * 40 * U * float(want)


def test_linear_gradients_by_differences():
    # central differences of f(h) = sum(dy * y(theta + h v)) in f32: step h = 2^-8, truncation ~ h^2, noise ~ 2^-24 * |f| / h
    gen = torch.Generator().manual_seed(11)
    leaves, dy = linear_case(33, 24, 20, "f32", "gelu", True, False, 0, 11)
    x, w, b, _ = leaves
    y = rows.linear(x, w, b, act=nn.GELU())
    grads = torch.autograd.grad(y, (x, w, b), dy)
    h = 2.0 ** -8
    for k, t in enumerate((x, w, b)):
        v = torch.randn(t.shape, generator=gen).to(DEV)
        v /= v.norm()
        args = [a.detach() for a in (x, w, b)]
        f = []
        for sign in (1, -1):
            moved = list(args)
            moved[k] = args[k] + sign * h * v
            f.append(float((rows.linear(*moved, act=nn.GELU()).double() * dy.double()).sum()))
        slope = float((grads[k].double() * v.double()).sum())
        terms = float(dy.double().abs().sum())
        assert abs((f[0] - f[1]) / (2 * h) - slope) <= 2 * h * h * terms + 64 * U * terms / h


@pytest.mark.parametrize("act", ["tanh", "sigmoid", "gelu", "gelu_tanh", "silu", "relu"])
def test_linear_bf16_gradients_cost_one_rounding(act):
    # dx and dw are rounded once as results and their operand dz once: independent errors of equal size, sqrt(2) = 1.414 of one
    # rounding's in the root mean square.  Nothing else may be visible (bound 1.45: over 10^5 values the ratio itself is known to 1 %)
    leaves, dy = linear_case(1024, 192, 256, "bf16", act, False, False, 0, 17)
    x, w = leaves[0], leaves[1]
    g = torch.autograd.grad(rows.linear(x, w, act=ACTS[act]), (x, w), dy)
    x64, w64, dy64 = x.detach().double().cpu(), w.detach().double().cpu(), dy.double().cpu()
    dz = dy64 * act64(x64 @ w64.t(), act)[1]
    for got, want in zip(g, (dz @ w64, dz.t() @ x64)):
        one = float((want.bfloat16().double() - want).norm())
        assert float((got.double().cpu() - want).norm()) <= 1.45 * one


def test_linear_slopes_at_infinity_and_nan():
    # the slope's limits: 0 on one side, 1 (or 0: tanh, sigmoid) on the other; NaN stays NaN for the smooth ones
    inf = float("inf")
    for dt in ("bf16", "f32"):
        # x of 1 and 0 picks the bias alone: z = b
        x = torch.zeros(70, 8, device=DEV, dtype=DT[dt]).requires_grad_()
        w = torch.ones(16, 8, device=DEV, dtype=DT[dt])
        b = torch.tensor([inf, -inf, 3e38, -3e38, float("nan")] + [0.0] * 11, device=DEV, dtype=DT[dt]).requires_grad_()
        for act, hi, lo in (("relu", 1, 0), ("lrelu", 1, 0.2), ("tanh", 0, 0), ("sigmoid", 0, 0), ("gelu", 1, 0), ("gelu_tanh", 1, 0), ("silu", 1, 0)):
            for res in (None, torch.zeros(70, 16, device=DEV, dtype=DT[dt])):
                y = rows.linear(x, w, b, act=ACTS[act], residual=res)
                (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
                want = torch.tensor([hi, lo, hi, lo], dtype=torch.float64) * 70
                # slopes are taken at 100 at most: sigmoid's there is e^-100 = 3.7e-44, 70 rows of it 2.6e-42
                torch.testing.assert_close(db[:4].double().cpu(), want, rtol=2.0 ** -8, atol=3e-42)
                assert act in ("relu", "lrelu") or torch.isnan(db[4])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("act,lo", [("relu", 0.0), ("lrelu", 0.2)])
def test_linear_slopes_at_and_next_to_the_kink(act, lo, res, dt):
    # z = b where x is zero (the rows a batch is padded with): 0 counts as negative, as in torch; far below a half's least value
    # the sign of z still decides
    x = torch.zeros(70, 8, device=DEV, dtype=DT[dt])
    w = torch.ones(16, 8, device=DEV, dtype=DT[dt])
    z = [0.0, -0.0, 1e-8, -1e-8, 1e-20, -1e-20, 1e-30, -1e-30] + [0.0] * 8
    b = torch.tensor(z, device=DEV, dtype=DT[dt]).requires_grad_()
    r = torch.ones(70, 16, device=DEV, dtype=DT[dt]) if res else None
    y = rows.linear(x, w, b, act=ACTS[act], residual=r)
    (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
    want = torch.tensor([70.0 if v > 0 else 70 * lo for v in z], dtype=torch.float64)
    torch.testing.assert_close(db.double().cpu(), want, rtol=2.0 ** -8, atol=0)       # sums of 70 in f32, one rounding


def test_linear_partial_gradients():
    leaves, dy = linear_case(40, 32, 24, "bf16", "silu", True, False, 0, 12)
    full = torch.autograd.grad(rows.linear(leaves[0], leaves[1], leaves[2], act=nn.SiLU()), leaves[:3], dy)
    for k in range(3):
        args = [t.detach().requires_grad_(j == k) for j, t in enumerate(leaves[:3])]
        (g,) = torch.autograd.grad(rows.linear(*args, act=nn.SiLU()), args[k], dy)
        assert torch.equal(g, full[k])


def test_no_second_derivatives():
    x = torch.randn(5, 8, device=DEV, requires_grad=True)
    w = torch.randn(6, 8, device=DEV, requires_grad=True)
    for f in (lambda: rows.linear(x, w, act=nn.Tanh()), lambda: rows.layer_norm(x), lambda: rows.dropout(x, 0.5, 1)):
        dy = torch.ones_like(f()).requires_grad_()
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(f(), x, dy, create_graph=True)
        (g,) = torch.autograd.grad(f(), x, dy)
        assert not g.requires_grad


def test_second_derivatives_are_refused_not_zero():
    # the first derivative under create_graph=True has its value; differentiating it raises although dy itself is a constant
    x = torch.randn(5, 8, device=DEV, requires_grad=True)
    w = torch.randn(6, 8, device=DEV, requires_grad=True)
    v = torch.randn(8, device=DEV, requires_grad=True)
    for f, ts in ((lambda: rows.linear(x, w, act=nn.Tanh()), (x, w)), (lambda: rows.linear(x, w), (x, w)),
                  (lambda: rows.layer_norm(x, v), (x, v))):
        first = torch.autograd.grad(f().sum(), ts)
        kept = torch.autograd.grad(f().sum(), ts, create_graph=True)
        for a, b in zip(first, kept):
            assert torch.equal(a, b.detach())
            with pytest.raises(RuntimeError, match="not differentiable"):
                ((b ** 2).sum() + (x ** 2).sum() + (w ** 2).sum()).backward()
    # nothing to refuse where the gradient is a constant: dx of a product with frozen weights
    y = rows.linear(x, w.detach())
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert not g.requires_grad


def test_library_errors_keep_their_type():
    from srmi import _lib as L
    x = torch.empty((1, (1 << 22) + 8), device=DEV, dtype=torch.bfloat16)
    with pytest.raises(L.SrmiError, match="2\\^22"):
        rows.linear(x, torch.empty((1, (1 << 22) + 8), device=DEV, dtype=torch.bfloat16))


def test_linear_same_call_same_bits():
    for dt in ("bf16", "f32"):
        leaves, dy = linear_case(700, 320, 192, dt, "gelu", True, True, 0, 13)
        runs = []
        for _ in range(2):
            y = rows.linear(leaves[0], leaves[1], leaves[2], act=nn.GELU(), residual=leaves[3])
            runs.append([y] + list(torch.autograd.grad(y, leaves, dy)))
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_linear_leaves_neighbours_alone():
    # outputs are dense, but operands are slices of wider buffers: nothing outside them is written
    gen = torch.Generator().manual_seed(14)
    wide = make((30, 64), "bf16", gen)
    before = wide.clone()
    x = wide[:, 8:40].requires_grad_()
    w = make((24, 32), "bf16", gen).requires_grad_()
    y = rows.linear(x, w, act=nn.ReLU())
    torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert torch.equal(wide, before)


def test_linear_nonfinite_rows_stay_in_their_rows():
    gen = torch.Generator().manual_seed(15)
    for dt in ("bf16", "f32"):
        x, w = make((130, 72), dt, gen), make((70, 72), dt, gen)
        ref = rows.linear(x, w)
        bad = x.clone()
        bad[3, 5], bad[77, 0] = float("nan"), float("inf")
        got = rows.linear(bad, w)
        keep = torch.ones(130, dtype=torch.bool, device=DEV)
        keep[[3, 77]] = False
        assert torch.equal(got[keep], ref[keep]) and not torch.isfinite(got[~keep]).any()


# ---- layer norm ----------------------------------------------------------------------------------------------------------
def check_norm(x, w, b, dy, dt, pdt):
    c = x.shape[-1]
    y = rows.layer_norm(x, w, b, eps=1e-5)
    leaves = [t for t in (x, w, b) if t is not None and t.requires_grad]
    names = [k for k, t in zip("xwb", (x, w, b)) if t is not None and t.requires_grad]
    grads = dict(zip(names, torch.autograd.grad(y, leaves, dy)))
    x64, dy64 = x.detach().double().cpu().reshape(-1, c), dy.double().cpu().reshape(-1, c)
    w64 = w.detach().double().cpu() if w is not None else torch.ones(c, dtype=torch.float64)
    b64 = b.detach().double().cpu() if b is not None else torch.zeros(c, dtype=torch.float64)
    n = x64.shape[0]
    mean = x64.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(x64.var(1, unbiased=False, keepdim=True) + 1e-5)
    xh = (x64 - mean) * rstd
    s, sp, k = half_step(dt), half_step(pdt), c + 16
    big = x64.abs().amax(1, keepdim=True) * rstd                         # |x| in units of the deviation: what subtracting the mean loses
    exh = k * U * (big + xh.abs() * (1 + big) + xh.abs())                # mean, variance (through the mean) and rstd
    want = xh * w64 + b64
    e = w64.abs() * exh + 4 * U * (w64 * xh).abs() + 2 * U * want.abs()
    assert y.dtype == DT[dt] and y.is_contiguous()
    assert_within(y.reshape(-1, c), want, e * (1 + s) + s * want.abs() + TINY, "y")
    g = dy64 * w64
    G = g.abs().mean(1, keepdim=True)
    c2 = (g * xh).mean(1, keepdim=True)
    GA = (g * xh).abs().mean(1, keepdim=True)
    ec2 = k * U * GA + (g.abs() * exh).mean(1, keepdim=True)
    want = rstd * (g - g.mean(1, keepdim=True) - xh * c2)
    e = rstd * (k * U * (g.abs() + G + xh.abs() * c2.abs()) * (1 + big) + exh * c2.abs() + (xh.abs() + exh) * ec2)
    if "x" in grads:
        assert_within(grads["x"].reshape(-1, c), want, e * (1 + s) + s * want.abs() + TINY, "dx")
    if "w" in grads:
        want = (dy64 * xh).sum(0)
        e = (dy64.abs() * exh).sum(0) + (n + 16) * U * (dy64 * xh).abs().sum(0)
        assert_within(grads["w"], want, e * (1 + sp) + sp * want.abs() + TINY, "dw")
    if "b" in grads:
        want = dy64.sum(0)
        assert_within(grads["b"], want, (n + 16) * U * dy64.abs().sum(0) * (1 + sp) + sp * want.abs() + TINY, "db")


def norm_case(n, c, dt, pdt, affine, pitch, seed, lead=None):
    gen = torch.Generator().manual_seed(seed)
    shape = (lead or (n,)) + (c,)
    x = make(shape, dt, gen, 1.5, pitch=pitch)
    x = (x + 0.75).detach() if not pitch else x
    w = (1 + make((c,), pdt, gen, 0.2)).requires_grad_() if affine else None
    b = make((c,), pdt, gen, 0.2).requires_grad_() if affine else None
    return x.requires_grad_(), w, b, make(shape, dt, gen, pitch=pitch)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("c", [1, 2, 5, 8, 16, 24, 64, 65, 128, 136, 256, 300, 512, 771, 1024, 1025, 1032, 2048, 2052, 2056, 4099, 8192, 20000])
def test_norm_widths(c, dt):
    for n in (1, 37):
        check_norm(*norm_case(n, c, dt, dt, True, 0, c + n), dt, dt)


# a row per workgroup, and more rows than workgroups: every sum is taken again and again in the same shared memory
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,c,pitch", [(1300, 4096, 0), (1100, 2049, 7), (700, 8191, 0), (600, 8192, 8), (2100, 8193, 0)])
def test_norm_many_wide_rows(n, c, pitch, dt):
    check_norm(*norm_case(n, c, dt, "f32", True, pitch, n + c), dt, "f32")


@pytest.mark.parametrize("dt,pdt", [("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("pitch", [0, 3, 8])
def test_norm_forms(dt, pdt, affine, pitch):
    for n, c in ((5, 96), (1111, 64), (3000, 33)):
        check_norm(*norm_case(n, c, dt, pdt, affine, pitch, n + pitch), dt, pdt)


def test_norm_empty_rows_and_leading_axes():
    for dt in ("bf16", "f32"):
        check_norm(*norm_case(0, 32, dt, dt, True, 0, 1), dt, dt)
        check_norm(*norm_case(None, 40, dt, dt, True, 0, 2, lead=(2, 3, 5)), dt, dt)
        x = torch.randn(40, device=DEV).to(DT[dt])                          # a single row without leading axes
        torch.testing.assert_close(rows.layer_norm(x), rows.layer_norm(x[None])[0], rtol=0, atol=0)


def test_norm_weight_or_bias_alone():
    gen = torch.Generator().manual_seed(3)
    x, w = make((9, 48), "f32", gen), make((48,), "f32", gen)
    y0 = rows.layer_norm(x)
    torch.testing.assert_close(rows.layer_norm(x, weight=w), y0 * w, rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(rows.layer_norm(x, bias=w), y0 + w, rtol=1e-6, atol=1e-6)
    b = w.clone().requires_grad_()
    y = rows.layer_norm(x, bias=b)
    (g,) = torch.autograd.grad(y, b, torch.ones_like(y))
    assert torch.equal(g, torch.full_like(g, 9.0))


def test_norm_constant_and_offset_rows():
    # a constant row has variance 0: xh = 0 exactly; a large common offset must not eat the deviations (two-pass variance)
    x = torch.full((4, 256), 3.0, device=DEV)
    assert torch.equal(rows.layer_norm(x), torch.zeros_like(x))
    gen = torch.Generator().manual_seed(4)
    d = torch.randint(-8, 9, (5, 256), generator=gen).double()
    x = (d + 2.0 ** 14).float().to(DEV)                                     # exact in f32
    want = (d - d.mean(1, keepdim=True)) / torch.sqrt(d.var(1, unbiased=False, keepdim=True) + 1e-5)
    assert float((rows.layer_norm(x).double().cpu() - want).abs().max()) <= 256 * U * 2.0 ** 14 * 2


def test_norm_same_call_same_bits_and_eps():
    x, w, b, dy = norm_case(5000, 192, "bf16", "bf16", True, 0, 5)
    runs = []
    for _ in range(2):
        y = rows.layer_norm(x, w, b, eps=0.5)
        runs.append([y] + list(torch.autograd.grad(y, (x, w, b), dy)))
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    x64 = x.detach().double()
    want = (x64 - x64.mean(1, keepdim=True)) / torch.sqrt(x64.var(1, unbiased=False, keepdim=True) + 0.5) * w.double() + b.double()
    assert float((runs[0][0].double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


# ---- dropout -------------------------------------------------------------------------------------------------------------
def philox(n, seed, offset):
    """word i % 4 of the Philox4x32-10 block with counter (i // 4, offset) and key seed, in Python integers"""
    out, m = [], 0xFFFFFFFF
    for block in range((n + 3) // 4):
        c = [block & m, block >> 32, offset & m, offset >> 32]
        k0, k1 = seed & m, seed >> 32
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k0, b & m, (a >> 32) ^ c[3] ^ k1, a & m]
            k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
        out += c
    return torch.tensor(out[:n], dtype=torch.float64)


def test_philox_known_answers():
    # the published vector of Philox4x32-10 for counter and key zero
    assert [int(v) for v in philox(4, 0, 0)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 255, 2049])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_mask_and_values(n, p, dt):
    gen = torch.Generator().manual_seed(n)
    seed, offset = 0xDEADBEEF12345678, (1 << 40) + 17
    keep = philox(n, seed, offset) >= math.floor(p * 2 ** 32)
    s = half_step(dt)
    for res in (False, True):
        for shift in (0, 1):                                                # shift 1: off the 16-byte boundary
            x = make((n + shift,), dt, gen)[shift:].requires_grad_()
            r = make((n + shift,), dt, gen)[shift:].requires_grad_() if res else None
            y = rows.dropout(x, p, seed, offset, residual=r)
            scaled = torch.where(keep, x.detach().double().cpu() * (1 / (1 - p) if p < 1 else 0.0), torch.zeros(n, dtype=torch.float64))
            want = scaled + (r.detach().double().cpu() if res else 0)
            assert_within(y, want, 4 * U * (scaled.abs() + want.abs()) + s * want.abs() + TINY, "y")
            dy = make((n,), dt, gen)
            g = torch.autograd.grad(y, [x] + ([r] if res else []), dy)
            want = torch.where(keep, dy.double().cpu() * (1 / (1 - p) if p < 1 else 0.0), torch.zeros(n, dtype=torch.float64))
            assert_within(g[0], want, 4 * U * want.abs() + s * want.abs() + TINY, "dx")
            assert not res or torch.equal(g[1], dy)


def test_dropout_drops_what_is_not_finite():
    x = torch.full((4096,), float("nan"), device=DEV)
    x[::2] = float("inf")
    y = rows.dropout(x, 0.5, 7)
    keep = philox(4096, 7, 0) >= 2 ** 31
    assert torch.equal(y.cpu()[~keep], torch.zeros(int((~keep).sum()))) and not torch.isfinite(y.cpu()[keep]).any()
    assert torch.equal(rows.dropout(x, 1.0, 7), torch.zeros_like(x))


def test_dropout_rate_and_streams_differ():
    x = torch.ones(1 << 20, device=DEV)
    a, b, c = (rows.dropout(x, 0.25, s, o) for s, o in ((1, 0), (1, 1), (2, 0)))
    # kept counts are binomial: 6 standard deviations of sqrt(n p q)
    assert abs(int((a != 0).sum()) - 0.75 * 2 ** 20) <= 6 * math.sqrt(2 ** 20 * 0.1875)
    for u, v in ((a, b), (a, c), (b, c)):
        agree = int(((u != 0) == (v != 0)).sum())
        assert abs(agree - 0.625 * 2 ** 20) <= 6 * math.sqrt(2 ** 20 * 0.625 * 0.375)


def test_dropout_device_counter_and_its_guard():
    x = torch.randn(1000, device=DEV, requires_grad=True)
    rng = torch.tensor([11, 5], dtype=torch.int64, device=DEV)
    y = rows.dropout(x, 0.3, rng)
    assert torch.equal(y, rows.dropout(x, 0.3, 11, 5))
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert torch.equal(rows.dropout(x.detach(), 0.3, rng), rows.dropout(x.detach(), 0.3, 11, 6))


def test_dropout_module():
    m = rows.Dropout(0.5, seed=3)
    x = torch.randn(64, 32, device=DEV)
    a, b = m(x), m(x)
    assert m.calls == 2 and torch.equal(a, rows.dropout(x, 0.5, 3, 1)) and torch.equal(b, rows.dropout(x, 0.5, 3, 2))
    assert torch.equal(m(x, residual=x), rows.dropout(x, 0.5, 3, 3, residual=x))
    m.eval()
    assert m(x) is x and torch.equal(m(x, residual=x), x + x)


# ---- refusals on device tensors ------------------------------------------------------------------------------------------
def test_refusals():
    x, w = torch.randn(4, 8, device=DEV), torch.randn(6, 8, device=DEV)
    for bad in (lambda: rows.linear(x, w.bfloat16()), lambda: rows.linear(x.double(), w.double()), lambda: rows.linear(x.half(), w.half()),
                lambda: rows.layer_norm(x, torch.ones(8, device=DEV, dtype=torch.bfloat16)), lambda: rows.dropout(x.long(), 0.1, 0),
                lambda: rows.layer_norm(x.bfloat16(), torch.ones(8, device=DEV), torch.ones(8, device=DEV, dtype=torch.bfloat16)),
                lambda: rows.dropout(x, 0.1, torch.zeros(2, device=DEV))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: rows.linear(x, w[:, :4]), lambda: rows.linear(x, w[0]), lambda: rows.linear(x, w, torch.zeros(8, device=DEV)),
                lambda: rows.linear(x, w, residual=torch.zeros(1, 6, device=DEV)), lambda: rows.layer_norm(x, torch.ones(4, device=DEV)),
                lambda: rows.layer_norm(x, eps=-1.0), lambda: rows.layer_norm(x, eps=float("nan")), lambda: rows.layer_norm(x[:, :0]),
                lambda: rows.dropout(x, 1.5, 0), lambda: rows.dropout(x, 0.1, -1), lambda: rows.dropout(x, 0.1, 1 << 64),
                lambda: rows.dropout(x, 0.1, 0, 1.5), lambda: rows.dropout(x, 0.1, 0, residual=x[:2]), lambda: rows.dropout(x, float("nan"), 0),
                lambda: rows.dropout(x, 0.1, torch.zeros(2, device=DEV, dtype=torch.int64), 3),
                lambda: rows.layer_norm(torch.tensor(1.0, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rows.linear(x, w.cpu())
    with pytest.raises(NotImplementedError):
        rows.linear(x, w, act=nn.PReLU().to(DEV))


# ---- a run of them together ----------------------------------------------------------------------------------------------
def _mixer(t, p, conv_in=None):
    h = rows.layer_norm(t, p["g"], p["b"])
    h = rows.linear(h, p["w1"], p["b1"], act=nn.GELU())
    h = rows.linear(h, p["w2"], p["b2"])
    return rows.dropout(h, 0.2, 99, 4, residual=t)


def _mixer64(t, p):
    c = t.shape[-1]
    m = t.mean(-1, keepdim=True)
    h = (t - m) / torch.sqrt(((t - m) ** 2).mean(-1, keepdim=True) + 1e-5) * p["g"] + p["b"]
    h = nn.functional.gelu(h @ p["w1"].t() + p["b1"]) @ p["w2"].t() + p["b2"]
    keep = (philox(t.numel(), 99, 4) >= math.floor(0.2 * 2 ** 32)).double().reshape(t.shape)
    return t + h * keep / 0.8


def _mixer_params(c, hid, dt, gen):
    p = {"g": 1 + make((c,), dt, gen, 0.1), "b": make((c,), dt, gen, 0.1), "w1": make((hid, c), dt, gen, c ** -0.5), "b1": make((hid,), dt, gen, 0.1),
         "w2": make((c, hid), dt, gen, hid ** -0.5), "b2": make((c,), dt, gen, 0.1)}
    return {k: v.requires_grad_() for k, v in p.items()}


@pytest.mark.parametrize("dt,tol", [("f32", 2e-5), ("bf16", 0.04)])
def test_channel_mixer(dt, tol):
    # chained roundings: about a dozen of half a step each, over sums of O(1) terms - relative to the largest value
    gen = torch.Generator().manual_seed(21)
    t = make((2, 5, 7, 64), dt, gen).requires_grad_()
    p = _mixer_params(64, 160, dt, gen)
    y = _mixer(t, p)
    dy = make(tuple(t.shape), dt, gen)
    got = [y] + list(torch.autograd.grad(y, [t] + list(p.values()), dy))
    t64 = t.detach().double().cpu().requires_grad_()
    p64 = {k: v.detach().double().cpu().requires_grad_() for k, v in p.items()}
    y64 = _mixer64(t64, p64)
    want = [y64.detach()] + list(torch.autograd.grad(y64, [t64] + list(p64.values()), dy.double().cpu()))
    for a, b in zip(got, want):
        assert float((a.double().cpu() - b).abs().max()) <= tol * float(b.abs().max())


def test_mixer_between_convolutions():
    # the operators on a channels-last map between two fused convs of this package: no copies, gradients reach the first conv
    torch.manual_seed(22)
    gen = torch.Generator().manual_seed(22)
    c1, c2 = nn.Conv2d(3, 32, 3, padding=1).to(DEV), nn.Conv2d(32, 3, 3, padding=1).to(DEV)
    p = _mixer_params(32, 96, "f32", gen)
    img = torch.randn(2, 3, 9, 11, generator=gen).to(DEV)
    feat = AG.fused_conv(img, c1, None, nn.ReLU())
    t = feat.permute(0, 2, 3, 1)
    assert t.is_contiguous()
    out = AG.fused_conv(_mixer(t, p).permute(0, 3, 1, 2), c2, None, None)
    params = [c1.weight, c2.weight] + list(p.values())
    got = [out] + list(torch.autograd.grad(out.square().mean(), params))
    d1, d2 = nn.Conv2d(3, 32, 3, padding=1).double(), nn.Conv2d(32, 3, 3, padding=1).double()
    d1.load_state_dict({k: v.double().cpu() for k, v in c1.state_dict().items()})
    d2.load_state_dict({k: v.double().cpu() for k, v in c2.state_dict().items()})
    p64 = {k: v.detach().double().cpu().requires_grad_() for k, v in p.items()}
    f64 = torch.relu(d1(img.double().cpu())).permute(0, 2, 3, 1)
    o64 = d2(_mixer64(f64, p64).permute(0, 3, 1, 2))
    want = [o64.detach()] + list(torch.autograd.grad(o64.square().mean(), [d1.weight, d2.weight] + list(p64.values())))
    for a, b in zip(got, want):
        assert float((a.double().cpu() - b).abs().max()) <= 1e-4 * float(b.abs().max())


def test_modules_train_together():
    torch.manual_seed(23)
    net = nn.Sequential(rows.LayerNorm(48), rows.Linear(48, 96, act=nn.SiLU()), rows.Linear(96, 48), rows.Dropout(0.1, seed=1)).to(DEV)
    x = torch.randn(6, 10, 48, device=DEV)
    net(x).square().mean().backward()
    assert all(q.grad is not None and torch.isfinite(q.grad).all() and float(q.grad.abs().max()) > 0 for q in net.parameters())


# ---- streams and graphs --------------------------------------------------------------------------------------------------
def _step(t, p, rng):
    h = rows.layer_norm(t, p["g"], p["b"])
    h = rows.linear(h, p["w1"], p["b1"], act=nn.GELU())
    h = rows.linear(h, p["w2"], p["b2"])
    return rows.dropout(h, 0.2, rng, residual=t)


def test_training_on_two_streams_at_once():
    gen = torch.Generator().manual_seed(30)
    jobs = []
    for i in range(2):
        p = _mixer_params(128, 320, "f32", gen)
        jobs.append((make((2000 + i, 128), "f32", gen).requires_grad_(), p, make((2000 + i, 128), "f32", gen)))

    def job(t, p, dy):
        y = rows.dropout(rows.linear(rows.linear(rows.layer_norm(t, p["g"], p["b"]), p["w1"], p["b1"], act=nn.GELU()), p["w2"], p["b2"]), 0.2, 1, 2,
                         residual=t)
        return [y] + list(torch.autograd.grad(y, [t] + list(p.values()), dy))

    want = [job(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for j, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(job(*j))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_two_streams_at_once():
    gen = torch.Generator().manual_seed(31)
    p = {k: v.detach() for k, v in _mixer_params(256, 512, "bf16", gen).items()}
    ts = [make((4096, 256), "bf16", gen) for _ in range(2)]
    want = [_mixer(t, p) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _mixer(ts[i], p)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_captured_graphs_replayed_in_turn():
    # forward and backward in one capture (fresh leaves, autograd.grad); two graphs replayed back to back on two streams must not
    # share scratch memory; the device counter moves between replays, so every replay draws another mask
    gen = torch.Generator().manual_seed(32)
    graphs = []
    for i in range(2):
        p = _mixer_params(64, 160, "bf16", gen)
        t = make((300 + i, 64), "bf16", gen).requires_grad_()
        dy = make((300 + i, 64), "bf16", gen)
        rng = torch.tensor([5 + i, 0], dtype=torch.int64, device=DEV)
        warm = torch.cuda.Stream()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            y = _step(t, p, rng)
            torch.autograd.grad(y, [t] + list(p.values()), dy)
            del y
        torch.cuda.current_stream().wait_stream(warm)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _step(t, p, rng)
            outs = [y] + list(torch.autograd.grad(y, [t] + list(p.values()), dy))
        graphs.append((graph, outs, t, p, dy, rng))
    side = torch.cuda.Stream()
    for it in range(4):
        for graph, outs, t, p, dy, rng in graphs:
            rng[1] = it
            with torch.no_grad():
                t.mul_(0.9).add_(0.01)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        for graph, outs, t, p, dy, rng in graphs:
            q = {k: v.detach().requires_grad_() for k, v in p.items()}
            tt = t.detach().clone().requires_grad_()
            y = _step(tt, q, rng)
            want = [y] + list(torch.autograd.grad(y, [tt] + list(q.values()), dy))
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), it


def test_capture_refuses_leaves_of_a_living_eager_graph():
    x = torch.randn(80, 64, device=DEV, requires_grad=True)
    w = torch.randn(48, 64, device=DEV, requires_grad=True)
    for f in (lambda: rows.linear(x, w), lambda: rows.layer_norm(x), lambda: rows.dropout(x, 0.5, 1)):
        alive = f()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(graph):
                f()
        torch.cuda.synchronize()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = f()
        graph.replay()
        torch.cuda.synchronize()
        got = y.detach().clone()
        del y, graph
        assert torch.equal(got, f().detach())


def test_capture_refuses_leaves_behind_the_operands():
    # the leaf that an eager graph still refers to is not an operand itself: an operand was computed from it
    x = torch.randn(80, 64, device=DEV, requires_grad=True)
    w = torch.randn(48, 64, device=DEV, requires_grad=True)
    alive = x * 2.0
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            rows.layer_norm(rows.linear((x + 1.0).relu(), w.detach()))
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (g,) = torch.autograd.grad(rows.layer_norm(rows.linear((x + 1.0).relu(), w.detach())), x, torch.ones(80, 48, device=DEV))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    got = g.clone()
    del graph
    (want,) = torch.autograd.grad(rows.layer_norm(rows.linear((x + 1.0).relu(), w.detach())), x, torch.ones(80, 48, device=DEV))
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    # 2^31 + elements in x and y: rows at the far end are computed from their own data
    c, n = 512, (1 << 22) + 3000                                            # 2.15e9 elements, 4.3 GB in bf16
    x = torch.empty((n, c), dtype=torch.bfloat16, device=DEV)
    x[: n // 2] = 0
    x[n // 2:] = 1
    gen = torch.Generator().manual_seed(41)
    tail = make((3000, c), "bf16", gen)
    x[-3000:] = tail
    w, b = make((8, c), "bf16", gen, c ** -0.5), make((c,), "bf16", gen)
    # against 64 bits: another number of rows may split the sum over k elsewhere, so the short call's bits are not promised
    t64, w64 = tail.double().cpu(), w.double().cpu()
    want = t64 @ w64.t()
    assert_within(rows.linear(x, w)[-3000:], want, 2.0 ** -8 * want.abs() + 1.01 * (c + 8) * U * (t64.abs() @ w64.abs().t()) + TINY, "far rows")
    y = rows.layer_norm(x, b, b)
    assert torch.equal(y[-3000:], rows.layer_norm(tail, b, b))
    del y
    y = rows.dropout(x, 0.5, 3)
    first = (n - 3000) * c
    bits = []
    for i in (first, first + 4 * 1000, n * c - 4):                           # blocks past 2^29 counters, elements past 2^31
        m, blk = 0xFFFFFFFF, i // 4
        cc, k0, k1 = [blk & m, blk >> 32, 0, 0], 3, 0
        for _ in range(10):
            a_, b_ = 0xD2511F53 * cc[0], 0xCD9E8D57 * cc[2]
            cc = [(b_ >> 32) ^ cc[1] ^ k0, b_ & m, (a_ >> 32) ^ cc[3] ^ k1, a_ & m]
            k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
        bits.append((i, cc))
    flat, src = y.view(-1), x.view(-1)
    for i, cc in bits:
        keep = torch.tensor([v >= 2 ** 31 for v in cc])
        assert torch.equal(flat[i:i + 4].float().cpu(), torch.where(keep, 2 * src[i:i + 4].float().cpu(), torch.zeros(4)))


def test_backward_offsets_past_32_bits():
    # y, z and dy of more than 2^32 elements: everything but the last rows is zero, so the gradients are those of the last rows alone
    k, n, m, far = 8, 520, (1 << 23) + 1000, 3000                            # 4.36e9 elements, 8.7 GB in bf16
    gen = torch.Generator().manual_seed(43)
    x = torch.zeros((m, k), dtype=torch.bfloat16, device=DEV)
    x[-far:] = make((far, k), "bf16", gen)
    w = make((n, k), "bf16", gen, k ** -0.5)
    dy = torch.zeros((m, n), dtype=torch.bfloat16, device=DEV)
    dy[-far:] = make((far, n), "bf16", gen)
    leaves = x.requires_grad_(), w.requires_grad_()
    y = rows.linear(*leaves, act=nn.GELU())
    dx, dw = torch.autograd.grad(y, leaves, dy)
    xs, ws = x[-far:].detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    short = rows.linear(xs, ws, act=nn.GELU())
    dxs, dws = torch.autograd.grad(short, (xs, ws), dy[-far:])
    assert not y[:-far].any() and not dx[:-far].any()
    x64, w64, dy64 = x[-far:].detach().double().cpu(), w.detach().double().cpu(), dy[-far:].double().cpu()
    f, g = act64(x64 @ w64.t(), "gelu")
    # two roundings of the storage type on either side of a sum (dz, and the result) and the slope's own error, as in check_linear
    s = 2.0 ** -8
    dz = dy64 * g
    edz = s * dz.abs() + dy64.abs() * (0.8 * (2.0 ** -11 * (x64 @ w64.t()).abs() + 2.0 ** -25) + FN["bf16"] * (g.abs() + 0.01)) * (1 + s)
    for got, near, want, e, c in ((dx[-far:], dxs, dz @ w64, edz @ w64.abs(), n), (dw, dws, dz.t() @ x64, edz.t() @ x64.abs(), far)):
        bound = (e + (c + 8) * U * 2 * e / s) * (1 + s) + s * want.abs() + TINY
        assert_within(near, want, bound, "short")
        assert_within(got, want, bound, "far")
    del y, dy, dx, short
    c = 1024
    x = torch.ones(((1 << 21) + 1000, c), dtype=torch.bfloat16, device=DEV)  # 2.15e9 elements
    x[-far:] = make((far, c), "bf16", gen)
    v = make((c,), "bf16", gen).requires_grad_()
    dy = torch.zeros_like(x)
    dy[-far:] = make((far, c), "bf16", gen)
    x.requires_grad_()
    dx, dv = torch.autograd.grad(rows.layer_norm(x, v), (x, v), dy)
    xs = x[-far:].detach().clone().requires_grad_()
    dxs, dvs = torch.autograd.grad(rows.layer_norm(xs, v), (xs, v), dy[-far:])
    assert torch.equal(dx[-far:], dxs) and not dx[:-far].any()
    # dv: the same f32 terms in another order, rounded once
    d64, t64 = dy[-far:].double().cpu(), xs.detach().double().cpu()
    xh = (t64 - t64.mean(1, keepdim=True)) / torch.sqrt(t64.var(1, unbiased=False, keepdim=True) + 1e-5)
    want = (d64 * xh).sum(0)
    bound = (far + c + 64) * U * (d64.abs() * (xh.abs() + 1)).sum(0) * (1 + s) + s * want.abs() + TINY
    assert_within(dv, want, bound, "far dv")
    assert_within(dvs, want, bound, "near dv")


# ---- saved-tensor hooks --------------------------------------------------------------------------------------------------
def _columns_first(t):
    """an equal tensor whose last axis is not dense"""
    return t.detach().transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.detach().clone()


# the saved tensor comes back with another pitch (dense, from the host), or with columns that have to be copied
HOOKS = {"save_on_cpu": lambda: torch.autograd.graph.save_on_cpu(),
         "columns_first": lambda: torch.autograd.graph.saved_tensors_hooks(_columns_first, lambda t: t)}


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("n,c", [(100, 64), (7, 33), (3, 9000)])
def test_norm_backward_under_saved_tensor_hooks(n, c, hook, dt):
    x, w, b, dy = norm_case(n, c, dt, "f32", True, 32, n + c)
    want = torch.autograd.grad(rows.layer_norm(x, w, b), (x, w, b), dy)
    with HOOKS[hook]():
        y = rows.layer_norm(x, w, b)
        got = torch.autograd.grad(y, (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("bad", [lambda t: t[:1], lambda t: t.double(), lambda t: t.cpu()])
def test_norm_refuses_what_a_hook_changed(bad):
    x, w, b, dy = norm_case(20, 48, "f32", "f32", True, 0, 1)
    for k in range(3):                                                       # x, weight, statistics, in the order they are saved
        order = iter(range(3))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: bad(t.detach()) if next(order) == k else t.detach(), lambda t: t):
            y = rows.layer_norm(x, w, b)
        with pytest.raises(RuntimeError, match="saved-tensor hook handed back"):
            torch.autograd.grad(y, (x, w, b), dy)


# "none" and "gelu" keep nothing / the pre-activation, "relu" the output itself
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("act", ["none", "gelu", "relu"])
@pytest.mark.parametrize("M,K,N,pitch", [(100, 72, 40, 24), (5, 72, 40, 24), (60, 33, 21, 13)])
def test_linear_backward_under_saved_tensor_hooks(M, K, N, pitch, act, hook, dt):
    leaves, dy = linear_case(M, K, N, dt, act, True, False, pitch, M + K)

    def run():
        with HOOKS[hook]():
            return rows.linear(*leaves[:3], act=ACTS[act])
    check_linear(leaves, dy, dt, act, run=run)


@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("bad", [lambda t: t[:1], lambda t: t.double(), lambda t: t.cpu()])
def test_linear_refuses_what_a_hook_changed(bad, act):
    leaves, dy = linear_case(20, 48, 24, "f32", act, True, False, 0, 2)
    for k in range(3):                                                       # x, weight, and what the slope is taken from
        order = iter(range(3))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: bad(t.detach()) if next(order) == k else t.detach(), lambda t: t):
            y = rows.linear(*leaves[:3], act=ACTS[act])
        with pytest.raises(RuntimeError, match="saved-tensor hook handed back"):
            torch.autograd.grad(y, leaves[:3], dy)


def test_dropout_device_counter_under_saved_tensor_hooks():
    x = torch.randn(40, 33, device=DEV, requires_grad=True)
    rng = torch.tensor([11, 5], dtype=torch.int64, device=DEV)
    dy = torch.randn(40, 33, device=DEV)
    (want,) = torch.autograd.grad(rows.dropout(x, 0.3, 11, 5), x, dy)
    apart = torch.tensor([11, 0, 5, 0], device=DEV)[::2]                     # equal, not dense
    for unpack in (lambda t: t, lambda t: apart):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
            y = rows.dropout(x, 0.3, rng)
            (got,) = torch.autograd.grad(y, x, dy)
        assert torch.equal(got, want)
    for bad in (lambda t: t[:1], lambda t: t.cpu(), lambda t: t.int(), lambda t: t.float()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), bad):
            y = rows.dropout(x, 0.3, rng)
            with pytest.raises(RuntimeError, match="saved-tensor hook handed back"):
                torch.autograd.grad(y, x, dy)


# ---- transforms that the operators cannot follow ---------------------------------------------------------------------------
def test_tangents_are_refused_in_both_passes():
    import torch.autograd.forward_ad as fwAD
    x, w = torch.randn(5, 8, device=DEV), torch.randn(6, 8, device=DEV)
    with fwAD.dual_level():
        for f in (lambda t: rows.linear(t, w), lambda t: rows.layer_norm(t), lambda t: rows.dropout(t, 0.5, 1)):
            leaf = x.clone().requires_grad_()
            y = f(leaf)
            dy = fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):          # forward over reverse
                torch.autograd.grad(y, leaf, dy)
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(fwAD.make_dual(x, torch.ones_like(x)))


def test_recorders_are_refused_in_both_passes():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.randn(5, 8, device=DEV, requires_grad=True), torch.randn(6, 8, device=DEV)
    for f in (lambda t: rows.linear(t, w), lambda t: rows.layer_norm(t), lambda t: rows.dropout(t, 0.5, 1)):
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                with pytest.raises(NotImplementedError, match="traced"):
                    torch.jit.trace(f, (x.detach(),))
                with pytest.raises(NotImplementedError, match="traced"):
                    make_fx(f)(x.detach())
        y = f(x)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda dy: torch.autograd.grad(y, x, dy))(torch.ones_like(y))


def test_modes_that_watch_or_recompute_get_the_results():
    from functools import partial
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    from torch.utils.flop_counter import FlopCounterMode
    gen = torch.Generator().manual_seed(61)
    p = _mixer_params(64, 96, "f32", gen)
    t = make((50, 64), "f32", gen).requires_grad_()
    dy = make((50, 64), "f32", gen)

    def step(f):
        y = f(t)
        return [y] + list(torch.autograd.grad(y, [t] + list(p.values()), dy))

    want = step(lambda u: _mixer(u, p))
    with FlopCounterMode(display=False):
        got = step(lambda u: _mixer(u, p))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for policy in (CheckpointPolicy.MUST_SAVE, CheckpointPolicy.PREFER_RECOMPUTE):
        contexts = partial(create_selective_checkpoint_contexts, lambda ctx, op, *a, **k: policy)
        got = step(lambda u: checkpoint(lambda q: _mixer(q, p), u, use_reentrant=False, context_fn=contexts))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), policy


def test_compiled_programs_call_the_operators_outside_their_graphs():
    gen = torch.Generator().manual_seed(62)
    p = _mixer_params(64, 96, "f32", gen)
    t = make((50, 64), "f32", gen).requires_grad_()
    dy = make((50, 64), "f32", gen)

    def f(u):
        return _mixer(u * 2.0, p) + 1.0

    y = f(t)
    want = [y] + list(torch.autograd.grad(y, [t] + list(p.values()), dy))
    y = torch.compile(f, backend="aot_eager")(t)
    got = [y] + list(torch.autograd.grad(y, [t] + list(p.values()), dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_negated_views_are_written_out():
    # the imaginary part of a conjugate is a view of the unconjugated memory with its sign still to be turned
    gen = torch.Generator().manual_seed(63)

    def both(shape):
        t = make(shape, "f32", gen)
        return torch._neg_view(-t), t

    (xn, x), (wn, w), (bn, b), (rn, r), (gn, g) = (both(s) for s in ((9, 16), (24, 16), (24,), (9, 24), (16,)))
    assert xn.is_neg() and torch.equal(xn, x)
    assert torch.equal(rows.linear(xn, wn, bn, act=nn.Tanh(), residual=rn), rows.linear(x, w, b, act=nn.Tanh(), residual=r))
    assert torch.equal(rows.layer_norm(xn, gn, gn), rows.layer_norm(x, g, g))
    assert torch.equal(rows.dropout(rn, 0.25, 4, residual=rn), rows.dropout(r, 0.25, 4, residual=r))
    for f in (lambda t: rows.linear(t, w), lambda t: rows.layer_norm(t), lambda t: rows.dropout(t, 0.5, 1)):
        x_ = x.clone().requires_grad_()
        dn, d = both(tuple(f(x_).shape))
        assert torch.equal(*(torch.autograd.grad(f(x_), x_, v)[0] for v in (dn, d)))
    z = make((8, 2), "f32", gen)
    col = torch.view_as_complex(z)[:, None].conj().imag                      # [8, 1], in place for a row operator
    assert col.is_neg() and torch.equal(rows.linear(col, torch.ones(1, 1, device=DEV)), -z[:, 1:])


@pytest.mark.parametrize("reentrant", [True, False])
def test_dropout_under_activation_checkpointing(reentrant):
    # the recomputed pass must draw the forward's mask: with another one the gradients belong to a different function
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(40, 64, device=DEV, requires_grad=True)
    w = torch.randn(64, 64, device=DEV, requires_grad=True)
    dy = torch.randn(40, 64, device=DEV)
    free = [rows.Dropout(0.5), rows.Dropout(0.5)]
    seeded = rows.Dropout(0.5, seed=5)

    def step(block, through):
        torch.manual_seed(8)
        out = [through(block, x), through(block, x)]
        return out + [g for y in out for g in torch.autograd.grad(y, (x, w), dy, retain_graph=True)]

    def drawn(t):
        return free[1](rows.linear(free[0](t), w, act=nn.GELU()))

    def stepped(t):
        return seeded(rows.linear(seeded(t, offset=11), w, act=nn.GELU()), offset=12)

    def counted(t):
        return rows.linear(seeded(t), w, act=nn.GELU())

    def again(block, t):
        return checkpoint(block, t, use_reentrant=reentrant)

    if reentrant:                                                            # that form supports .backward() alone
        def step(block, through):
            torch.manual_seed(8)
            out = [through(block, x), through(block, x)]
            x.grad = w.grad = None
            ((out[0] + 2 * out[1]) * dy).sum().backward()
            return [o.detach() for o in out] + [x.grad, w.grad]

    for block in (drawn, stepped):
        want = step(block, lambda f, t: f(t))
        assert all(torch.equal(a, b) for a, b in zip(step(block, again), want))
    assert seeded.calls == 0
    y = again(counted, x)
    with pytest.raises(RuntimeError, match="recomputed inside a backward pass"):
        y.sum().backward()
    assert seeded.calls == 1


def test_dropout_modules_differ_and_resume():
    x = torch.randn(64, 32, device=DEV)
    a, b = rows.Dropout(0.5), rows.Dropout(0.5)
    assert not torch.equal(a(x), b(x)) and not torch.equal(a(x), a(x))
    m = rows.Dropout(0.5, seed=3)
    m(x)
    resumed = rows.Dropout(0.5, seed=3)
    resumed.load_state_dict(m.state_dict())
    assert torch.equal(m(x), resumed(x)) and torch.equal(m(x, offset=1), rows.dropout(x, 0.5, 3, 1)) and m.calls == 2
    rng = torch.tensor([3, 1], device=DEV)
    assert torch.equal(a(x, rng=rng), rows.dropout(x, 0.5, 3, 1))
    with pytest.raises(ValueError, match="no other offset"):
        m(x, rng=rng, offset=2)
    net = torch.compile(lambda t: a(t * 2.0) + 1.0, backend="aot_eager")
    torch.manual_seed(9)
    got = net(x)
    torch.manual_seed(9)
    assert torch.equal(got, a(x * 2.0) + 1.0)


# ---- the C entry points ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("c", [8, 4096, 9000])
def test_norm_backward_of_no_rows(c, dt):
    import ctypes as C

    from srmi import _lib as L
    lib, n = L.load(), C.c_size_t(0)
    d = L.NormDesc(0, c, L.F32 if dt == "f32" else L.BF16, L.F32, 1e-5, c, c)
    L.check(lib.srmi_layer_norm_workspace_bytes(C.byref(d), C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device=DEV)
    dx, dw, db = (torch.full((c,), 7.0, device=DEV) for _ in range(3))
    stream = torch.cuda.current_stream().cuda_stream
    L.check(lib.srmi_layer_norm_bwd(C.byref(d), None, None, None, None, None, dx.data_ptr(), None, None, None, 0, stream))
    L.check(lib.srmi_layer_norm_bwd(C.byref(d), None, None, None, None, None, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), n.value, stream))
    torch.cuda.synchronize()
    assert not dw.any() and not db.any() and bool((dx == 7).all())           # sums of nothing; no row of dx to write


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_norm_widest_rows(dt):
    # the columns of dw and db together are 2^26, one launch adds them up
    c = 1 << 25
    x = torch.randn((2, c), device=DEV).to(DT[dt]).requires_grad_()
    w = torch.ones(c, device=DEV, dtype=DT[dt]).requires_grad_()
    b = torch.zeros(c, device=DEV, dtype=DT[dt]).requires_grad_()
    dy = (torch.arange(2 * c, device=DEV) % 251 - 125).reshape(2, c).to(DT[dt])
    y = rows.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x64, dy64 = x.detach().double(), dy.double()
    mean = x64.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x64 - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    xh = (x64 - mean) * rstd
    s, e = half_step(dt), (c / 256 + 64) * U                                 # 256 lanes: c / 256 sums one after another, |x| and deviation alike
    for got, want, big in ((y, xh, xh.abs() + 1), (dw, (dy64 * xh).sum(0), (dy64.abs() * (xh.abs() + 1)).sum(0)), (db, dy64.sum(0), dy64.abs().sum(0)),
                           (dx, rstd * (dy64 - dy64.mean(1, keepdim=True) - xh * (dy64 * xh).mean(1, keepdim=True)), 250 * (xh.abs() + 1))):
        assert float(((got.double() - want).abs() - e * big * (1 + s) - s * want.abs()).max()) <= 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_linear_most_features(dt):
    # 2^22 outputs of few rows: the bias gradient's strips of columns are one axis of the grid
    m, n = 3, 1 << 22
    x = torch.tensor([[1.0], [2.0], [-1.0]], device=DEV, dtype=DT[dt]).requires_grad_()
    w = (torch.arange(n, device=DEV) % 15 - 7).to(DT[dt])[:, None].requires_grad_()
    b = torch.zeros(n, device=DEV, dtype=DT[dt]).requires_grad_()
    dy = (torch.arange(m * n, device=DEV) % 7 - 3).reshape(m, n).to(DT[dt])
    y = rows.linear(x, w, b, act=nn.ReLU())
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    z = x.detach().double() * w.detach().double()[:, 0]                      # small integers: exact, but for the sum over n
    dz = dy.double() * (z > 0)
    assert torch.equal(y.double(), z.clamp(min=0)) and torch.equal(db.double(), dz.sum(0))
    assert torch.equal(dw.double(), (dz * x.detach().double()).sum(0)[:, None])
    want = (dz * w.detach().double()[:, 0]).sum(1, keepdim=True)
    assert bool(((dx.double() - want).abs() <= half_step(dt) * want.abs()).all())    # integers below 2^24 in every partial sum


def test_linear_more_tiles_than_a_launch_takes():
    # 2^30 rows of one column are 2^24 tiles of 64 rows and 256 threads: 2^32 threads, one too many for one launch
    m, far = (1 << 30) + 1000, 1000
    x = (torch.arange(m, device=DEV, dtype=torch.int32) % 17 - 8).float()[:, None].requires_grad_()
    w = torch.full((1, 1), 0.5, device=DEV, requires_grad=True)
    b = torch.ones(1, device=DEV, requires_grad=True)
    dy = torch.zeros(m, 1, device=DEV)
    dy[:far] = 3.0
    dy[-far:] = (torch.arange(far, device=DEV) % 7 - 3).float()[:, None]
    y = rows.linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():                                                    # halves and small integers: every sum is exact
        assert torch.equal(y, x * 0.5 + 1) and torch.equal(dx, dy * 0.5)
        ends = torch.cat((x[:far], x[-far:])), torch.cat((dy[:far], dy[-far:]))
        assert float(dw) == float((ends[0] * ends[1]).sum()) and float(db) == float(ends[1].sum())
    del x, y, dy, dx
    # the tiles of the DMA, residual and all: 128 rows each, more than 2^23 of them
    period, times = 1 << 15, (1 << 15) + 3
    gen = torch.Generator().manual_seed(72)
    x0, w, b, r0 = make((period, 8), "bf16", gen), make((8, 8), "bf16", gen), make((8,), "bf16", gen), make((period, 8), "bf16", gen)
    x, r = x0.repeat(times, 1).requires_grad_(), r0.repeat(times, 1)
    x0.requires_grad_()
    y0, y = rows.linear(x0, w, b, act=nn.GELU(), residual=r0), rows.linear(x, w, b, act=nn.GELU(), residual=r)
    assert bool((y.detach().view(times, period, 8) == y0.detach()).all())
    (dx0,), (dx,) = torch.autograd.grad(y0, x0, r0), torch.autograd.grad(y, x, r)
    assert bool((dx.view(times, period, 8) == dx0).all())


# ---- every tile kernel, with what its epilogue can do ------------------------------------------------------------------------
def check_linear_64(leaves, dy, dt, act):
    """check_linear with the 64-bit products on the GPU, for sizes that take the large tiles; the same bounds"""
    x, w, b, r = leaves
    (M, K), N = x.shape, w.shape[0]
    wanted = [t for t in leaves if t is not None]
    y = rows.linear(x, w, b, act=ACTS[act], residual=r)
    grads = dict(zip([k for k, t in zip("xwbr", leaves) if t is not None], torch.autograd.grad(y, wanted, dy)))
    with torch.no_grad():
        x64, w64, dy64 = x.double(), w.double(), dy.double()
        b64 = b.double() if b is not None else torch.zeros(N, dtype=torch.float64, device=DEV)
        wt = w64.t().contiguous()
        z = x64 @ wt + b64
    f, g = act64(z, act)
    s, fn = half_step(dt), FN[dt]
    with torch.no_grad():
        ez = (K + 8) * U * (x64.abs() @ wt.abs() + b64.abs())
        out = f + (r.double() if r is not None else 0)
        ey = LIP[act] * ez + fn * (f.abs() + 0.01 * z.abs()) + 2 * U * out.abs() + s * out.abs() + TINY

        def within(got, want, bound, what):
            assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
            assert float(((got.double() - want).abs() - bound).max()) <= 0, what

        within(y, out, ey + s * ey, "y")
        dz = dy64 * g
        zq = (2.0 ** -11 * z.abs() + 2.0 ** -25 if dt == "bf16" else 0) + ez
        edz = dy64.abs() * (CURV[act] * zq + fn * (g.abs() + 0.01) * (act != "none"))
        if act in ("relu", "lrelu"):
            edz = edz + dy64.abs() * (z.abs() <= ez)
        edz_q = edz + (s if act != "none" else 0) * (dz.abs() + edz)
        if b is not None:
            want = dz.sum(0)
            within(grads["b"], want, (edz.sum(0) + (M + 8) * U * dz.abs().sum(0)) * (1 + s) + s * want.abs() + TINY, "db")
        for name, p, q, ep, n in (("x", dz, w64, edz_q, N), ("w", dz.t().contiguous(), x64, edz_q.t().contiguous(), M)):
            want = p @ q
            e = ep @ q.abs() + (n + 8) * U * ((p.abs() + ep) @ q.abs())
            within(grads[name], want, e * (1 + s) + s * want.abs() + TINY, "d" + name)
        assert r is None or torch.equal(grads["r"], dy)


# bf16 tiles of 128 x 128 with 64 k per stage, not split: prompt-sized products, all three of them
@pytest.mark.parametrize("act,bias,res", [("none", False, False), ("gelu", True, True), ("relu", True, False), ("silu", False, True)])
def test_linear_unsplit_128_tiles(act, bias, res):
    leaves, dy = linear_case(2040, 2200, 2056, "bf16", act, bias, res, 0, 81)
    check_linear_64(leaves, dy, "bf16", act)


# 256 x 256 in the forward product
@pytest.mark.parametrize("act,bias,res", [("gelu", True, True), ("lrelu", True, False), ("relu", False, True), ("tanh", False, False)])
def test_linear_256_tiles_with_epilogue(act, bias, res):
    leaves, dy = linear_case(3590, 520, 3608, "bf16", act, bias, res, 8, 82)
    check_linear_64(leaves, dy, "bf16", act)


# 32 x 128, not split: the forward of a wide head, its input gradient, and the weight gradient of a narrow one
@pytest.mark.parametrize("M,K,N", [(20, 2112, 33000), (20, 33000, 72), (500, 33000, 24)])
@pytest.mark.parametrize("act,bias,res", [("gelu", True, True), ("relu", True, False)])
def test_linear_unsplit_32_tiles(M, K, N, act, bias, res):
    leaves, dy = linear_case(M, K, N, "bf16", act, bias, res, 0, 83)
    check_linear_64(leaves, dy, "bf16", act)


# f32: tiles of 64 (unsplit and split) and of 128 (unsplit in the forward, split; dx and dw split), and the few-row kernels
@pytest.mark.parametrize("M,K,N", [(700, 96, 200), (700, 264, 200), (2900, 300, 2950), (1100, 2100, 1090), (16, 2950, 300), (24, 300, 1090)])
def test_linear_f32_products_keep_24_bits(M, K, N):
    # the per-element bound of check_linear grows with K until it no longer sees 16-bit operands; this one does (test_rows_cpu.py)
    leaves, dy = linear_case(M, K, N, "f32", "none", False, False, 0, 84)
    x, w = leaves[0], leaves[1]
    y = rows.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x64, w64, dy64 = x.detach().double(), w.detach().double(), dy.double()
    for got, a, b in ((y, x64, w64.t().contiguous()), (dx, dy64, w64), (dw, dy64.t().contiguous(), x64)):
        want = a @ b
        sigma = float(a.square().mean().sqrt() * b.square().mean().sqrt())
        err = float((got.detach().double() - want).square().mean().sqrt())
        assert err <= f32_product_rms(a.shape[1], sigma, float(want.square().mean().sqrt()))


class Guarded:
    """`n` bytes of 0xff (NaN in every storage type) with 64 KiB of a pattern on either side"""
    EDGE = 1 << 16

    def __init__(self, n):
        self.n, whole = n, 2 * self.EDGE + n
        self.buf = torch.full((whole,), 0xA5, dtype=torch.uint8, device=DEV)
        self.buf[self.EDGE:self.EDGE + n] = 0xFF

    def ptr(self):
        assert self.buf.data_ptr() % 256 == 0
        return self.buf.data_ptr() + self.EDGE

    def view(self, dt):
        return self.buf[self.EDGE:self.EDGE + self.n].view(dt)

    def intact(self):
        return bool((self.buf[:self.EDGE] == 0xA5).all()) and bool((self.buf[self.EDGE + self.n:] == 0xA5).all())


def _guarded(**sizes):
    return {k: Guarded(n) for k, n in sizes.items()}


def _check_guarded(bufs, written):
    torch.cuda.synchronize()
    for name, g in bufs.items():
        assert g.intact(), f"written past {name}"
    for name, dt in written.items():
        assert bool(torch.isfinite(bufs[name].view(dt).float()).all()), f"{name} is not written whole"


@pytest.mark.parametrize("M,K,N,dt,act", [(1, 1, 1, "bf16", "gelu"), (1, 1, 1, "f32", "gelu"), (17, 33, 5, "bf16", "relu"), (17, 33, 5, "f32", "silu"),
                                          (5, 4101, 35, "f32", "tanh"), (5, 4104, 35, "bf16", "tanh"), (63, 264, 41, "bf16", "gelu"), (20, 2112, 33001, "bf16", "none"),
                                          (300, 520, 203, "bf16", "gelu"), (301, 519, 203, "bf16", "gelu"), (500, 33000, 21, "bf16", "relu"),
                                          (2039, 2200, 2053, "bf16", "silu"), (3591, 520, 3603, "bf16", "gelu"), (1100, 2101, 1091, "f32", "none"),
                                          (2901, 300, 2950, "f32", "gelu"), (700, 96, 201, "f32", "lrelu"), (203, 5, 3, "f32", "sigmoid"), (203, 5, 3, "bf16", "gelu_tanh")])
def test_linear_writes_its_outputs_and_nothing_else(M, K, N, dt, act):
    import ctypes as C

    from srmi import _lib as L
    lib, n = L.load(), C.c_size_t(0)
    leaves, dy = linear_case(M, K, N, dt, act, True, True, 0, 85)
    x, w, b, r = (t.detach() for t in leaves)
    code, param = rows._act_of(ACTS[act])
    e = 2 if dt == "bf16" else 4
    d = L.LinearDesc(M, N, K, L.BF16 if dt == "bf16" else L.F32, code, param, 16, K, K, N, N)
    stream = torch.cuda.current_stream().cuda_stream
    L.check(lib.srmi_linear_workspace_bytes(C.byref(d), L.PASS_FWD, C.byref(n)))
    bufs = _guarded(y=M * N * e, z=M * N * e, ws=n.value)
    L.check(lib.srmi_linear_fwd(C.byref(d), x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), bufs["y"].ptr(), bufs["z"].ptr(), bufs["ws"].ptr(),
                                n.value, stream))
    kept = torch.float16 if dt == "bf16" else torch.float32
    _check_guarded(bufs, {"y": DT[dt], "z": kept})
    y = rows.linear(x, w, b, act=ACTS[act], residual=r)
    assert torch.equal(bufs["y"].view(DT[dt]), y.flatten())
    z = bufs["z"]
    L.check(lib.srmi_linear_workspace_bytes(C.byref(d), L.PASS_BWD, C.byref(n)))
    for wanted in ("dx dw db", "dx", "dw", "db", "dw db"):
        bufs = _guarded(dx=M * K * e, dw=N * K * e, db=N * e, ws=n.value)
        L.check(lib.srmi_linear_bwd(C.byref(d), x.data_ptr(), w.data_ptr(), z.ptr(), dy.data_ptr(),
                                    *(bufs[k].ptr() if k in wanted.split() else None for k in ("dx", "dw", "db")), bufs["ws"].ptr(), n.value, stream))
        _check_guarded(bufs, {k: DT[dt] for k in wanted.split()})
        for k in ("dx", "dw", "db"):
            assert k in wanted.split() or bool((bufs[k].view(torch.uint8) == 0xFF).all())


@pytest.mark.parametrize("dt,pdt", [("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 7), (37, 65), (1111, 257), (9, 1025), (600, 2049), (5, 8193), (700, 20001)])
def test_norm_writes_its_outputs_and_nothing_else(n, c, dt, pdt):
    import ctypes as C

    from srmi import _lib as L
    lib, size = L.load(), C.c_size_t(0)
    x, w, b, dy = norm_case(n, c, dt, pdt, True, 0, 86)
    x, w, b = x.detach(), w.detach(), b.detach()
    code = {"bf16": L.BF16, "f32": L.F32}
    e, pe = torch.finfo(DT[dt]).bits // 8, torch.finfo(DT[pdt]).bits // 8
    d = L.NormDesc(n, c, code[dt], code[pdt], 1e-5, c, c)
    stream = torch.cuda.current_stream().cuda_stream
    kept = _guarded(y=n * c * e, mean=n * 4, rstd=n * 4)
    L.check(lib.srmi_layer_norm_fwd(C.byref(d), x.data_ptr(), w.data_ptr(), b.data_ptr(), *(kept[k].ptr() for k in ("y", "mean", "rstd")), stream))
    _check_guarded(kept, {"y": DT[dt], "mean": torch.float32, "rstd": torch.float32})
    assert torch.equal(kept["y"].view(DT[dt]), rows.layer_norm(x, w, b).flatten())
    L.check(lib.srmi_layer_norm_workspace_bytes(C.byref(d), C.byref(size)))
    for wanted in ("dx dw db", "dx", "dw", "db"):
        bufs = _guarded(dx=n * c * e, dw=c * pe, db=c * pe, ws=size.value)
        L.check(lib.srmi_layer_norm_bwd(C.byref(d), x.data_ptr(), w.data_ptr(), kept["mean"].ptr(), kept["rstd"].ptr(), dy.data_ptr(),
                                        *(bufs[k].ptr() if k in wanted.split() else None for k in ("dx", "dw", "db")), bufs["ws"].ptr(), size.value, stream))
        _check_guarded(bufs, {k: DT[dt] if k == "dx" else DT[pdt] for k in wanted.split()})


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 5, 2047, 100003])
def test_dropout_writes_its_output_and_nothing_else(n, dt):
    from srmi import _lib as L
    lib, e = L.load(), 2 if dt == "bf16" else 4
    x = torch.ones(n, device=DEV, dtype=DT[dt])
    bufs = _guarded(y=n * e)
    L.check(lib.srmi_dropout(x.data_ptr(), x.data_ptr(), bufs["y"].ptr(), n, L.BF16 if dt == "bf16" else L.F32, 0.5, 1, 2, None,
                             torch.cuda.current_stream().cuda_stream))
    _check_guarded(bufs, {"y": DT[dt]})
    assert torch.equal(bufs["y"].view(DT[dt]), rows.dropout(x, 0.5, 1, 2, residual=x))


# ---- capture after warm-up runs on a side stream ------------------------------------------------------------------------------
def _block(dt):
    torch.manual_seed(90)
    return nn.Sequential(rows.LayerNorm(64), rows.Linear(64, 160, act=nn.GELU()), rows.Linear(160, 64)).to(DEV).to(DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_graphed_callables(dt):
    # the warm-up's last graph is still referred to while the capture runs: its leaves' nodes belong to the warm-up stream
    a, b = _block(dt), _block(dt)
    graphed = torch.cuda.make_graphed_callables(a, (torch.randn(300, 64, device=DEV, dtype=DT[dt], requires_grad=True),))
    for _ in range(4):
        x = torch.randn(300, 64, device=DEV, dtype=DT[dt])
        dy = torch.randn(300, 64, device=DEV, dtype=DT[dt])
        got, want = [], []
        for f, net, out in ((graphed, a, got), (b, b, want)):
            net.zero_grad(set_to_none=True)
            leaf = x.clone().requires_grad_()
            y = f(leaf)
            y.backward(dy)
            out += [y.detach().clone(), leaf.grad] + [p.grad.clone() for p in net.parameters()]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_captured_training_step_after_warm_up(dt):
    a, b = _block(dt), _block(dt)
    x, dy = (torch.randn(300, 64, device=DEV, dtype=DT[dt]) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            a.zero_grad(set_to_none=True)
            alive = a(x)
            alive.backward(dy)
    torch.cuda.current_stream().wait_stream(side)
    a.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = a(x)
        y.backward(dy)
    assert alive.grad_fn is not None
    for _ in range(4):
        x.copy_(torch.randn(300, 64, device=DEV))
        graph.replay()
        b.zero_grad(set_to_none=True)
        want = b(x)
        want.backward(dy)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(a.parameters(), b.parameters()))


def test_capture_refuses_operands_computed_on_the_default_stream():
    # the leaf's node belongs to a side stream, the operation between it and the captured call to the default one
    x = torch.randn(80, 64, device=DEV, requires_grad=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        alive = rows.layer_norm(x)
    torch.cuda.synchronize()
    h = x * 2.0
    for f in (lambda t: rows.linear(t, t), lambda t: rows.layer_norm(t), lambda t: rows.dropout(t, 0.5, 1)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(graph):
                f(h)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                                        # the leaf itself is fine
            f(x)
    assert alive.grad_fn is not None


@pytest.mark.parametrize("M", [8, 200])                                      # the f32 matrix instruction, and three bf16 planes
@pytest.mark.parametrize("e", [-148, -140, -133, -126, -120, -115, -110, -100, -60, 60, 100, 120])
def test_linear_f32_range(e, M):
    # x = hi + mid + lo has 24 bits unless the low plane ends at bf16's least step, 2^-133: off by half of that at most
    gen = torch.Generator().manual_seed(91)
    K, N = 40, 64
    x = (1 + torch.rand(M, K, generator=gen, dtype=torch.float64)) * (torch.randint(0, 2, (M, K), generator=gen) * 2 - 1)
    x = (x * 2.0 ** e).float()
    w = torch.randn(N, K, generator=gen)
    x64, w64 = x.double(), w.double()
    want = x64 @ w64.t()
    mag = x64.abs() @ w64.abs().t()
    bound = (K + 8) * U * mag + 2.0 ** -134 * (w64.abs().sum(1) + K)[None] + 2.0 ** -148
    assert_within(rows.linear(x.to(DEV), w.to(DEV)), want, bound, "y")
