"""CPU: refusals of the row operators - Python checks and the C ABI's validation, which comes before any launch."""
import ctypes as C

import pytest
import torch
import torch.nn as nn

from srmi import _lib as L
from srmi import rows


def test_cpu_tensors_are_refused():
    x, w = torch.randn(3, 8), torch.randn(5, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rows.linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rows.layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rows.dropout(x, 0.5, 1)


def test_non_tensors_are_refused():
    with pytest.raises(TypeError):
        rows.linear([1.0], torch.randn(1, 1))
    with pytest.raises(TypeError):
        rows.layer_norm(3.0)


def test_modules_refuse_what_they_cannot_run():
    with pytest.raises(NotImplementedError):
        rows.Linear(4, 4, act=nn.PReLU())
    with pytest.raises(NotImplementedError):
        rows.Linear(4, 4, act=nn.Hardtanh())
    with pytest.raises(NotImplementedError):
        rows.LayerNorm((4, 4))
    with pytest.raises(ValueError):
        rows.Dropout(1.5)
    lin, ref = rows.Linear(4, 3, act=nn.GELU()), nn.Linear(4, 3)
    assert list(lin.state_dict()) == list(ref.state_dict())
    assert list(rows.LayerNorm(8).state_dict()) == list(nn.LayerNorm(8).state_dict())


def test_struct_layout():
    assert C.sizeof(L.LinearDesc) == 8 + 6 * 4 + 4 * 8
    assert L.LinearDesc.ldx.offset == 32
    assert C.sizeof(L.NormDesc) == 8 + 4 * 4 + 2 * 8


def _lin(**kw):
    d = L.LinearDesc(4, 8, 16, L.F32, L.ACT_NONE, 0.0, 0, 16, 16, 8, 8)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("field,value", [("M", -1), ("N", -1), ("K", -2), ("M", L.ROWS_MAX + 1), ("dtype", 2), ("act", L.ACT_PRELU),
                                         ("act", L.ACT_ADD_RELU), ("act", 10), ("act", -1), ("ldx", 15), ("ldw", 0), ("ldr", 7), ("lddy", 3),
                                         ("ldr", -8), ("N", (1 << 22) + 1), ("K", (1 << 22) + 1)])
def test_linear_descriptor_refusals(field, value):
    lib, n = L.load(), C.c_size_t(0)
    d = _lin(**{field: value})
    assert lib.srmi_linear_workspace_bytes(C.byref(d), L.PASS_FWD, C.byref(n)) < 0
    assert lib.srmi_last_error() != b""
    big = 1 << 40
    assert lib.srmi_linear_fwd(C.byref(d), big, big, None, None, big, None, big, big, None) < 0
    assert lib.srmi_linear_bwd(C.byref(d), big, big, big, big, big, big, big, big, big, None) < 0


def test_linear_argument_refusals():
    lib, n = L.load(), C.c_size_t(0)
    d = _lin()
    assert lib.srmi_linear_workspace_bytes(None, 0, C.byref(n)) == -1
    assert lib.srmi_linear_workspace_bytes(C.byref(d), 2, C.byref(n)) == -1
    assert lib.srmi_linear_workspace_bytes(C.byref(d), 0, None) == -1
    big = 1 << 40
    for hole in range(3):                                                       # x, w, y
        a = [big, big, big]
        a[hole] = None
        assert lib.srmi_linear_fwd(C.byref(d), a[0], a[1], None, None, a[2], None, None, 0, None) == -1
    assert lib.srmi_linear_fwd(C.byref(d), big + 2, big, None, None, big, None, None, 0, None) == -1     # not on an element
    assert lib.srmi_linear_fwd(C.byref(_lin(ldr=0)), big, big, None, big, big, None, None, 0, None) == -1
    assert lib.srmi_linear_bwd(C.byref(d), big, big, None, None, big, big, big, None, 0, None) == -1     # no dy
    assert lib.srmi_linear_bwd(C.byref(_lin(act=L.ACT_GELU)), big, big, None, big, big, big, big, None, 0, None) == -1   # no z
    assert lib.srmi_linear_bwd(C.byref(d), None, big, None, big, None, big, None, big, 1 << 30, None) == -1     # dw without x
    assert lib.srmi_linear_bwd(C.byref(d), big, None, None, big, big, None, None, big, 1 << 30, None) == -1     # dx without w
    L.check(lib.srmi_linear_workspace_bytes(C.byref(_lin(act=L.ACT_GELU)), L.PASS_BWD, C.byref(n)))
    assert n.value > 0
    assert lib.srmi_linear_bwd(C.byref(_lin(act=L.ACT_GELU)), big, big, big, big, big, big, big, big, n.value - 1, None) == -1
    assert lib.srmi_linear_bwd(C.byref(_lin(act=L.ACT_GELU)), big, big, big, big, big, big, big, None, n.value, None) == -1
    assert lib.srmi_linear_bwd(C.byref(_lin(act=L.ACT_GELU)), big, big, big, big, big, big, big, big + 16, n.value, None) == -1
    assert lib.srmi_linear_fwd(C.byref(_lin(M=0)), None, None, None, None, None, None, None, 0, None) == 0     # nothing to do
    assert lib.srmi_linear_fwd(C.byref(_lin(N=0)), None, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(C=0), dict(C=-4), dict(dtype=5), dict(param_dtype=5), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(ldx=7), dict(lddy=7), dict(rows=L.ROWS_MAX + 1),
                                dict(C=L.NORM_MAX_C + 1, ldx=1 << 30, lddy=1 << 30)])
def test_norm_descriptor_refusals(kw):
    lib, n = L.load(), C.c_size_t(0)
    d = L.NormDesc(4, 8, L.F32, L.F32, 1e-5, 8, 8)
    for k, v in kw.items():
        setattr(d, k, v)
    big = 1 << 40
    assert lib.srmi_layer_norm_workspace_bytes(C.byref(d), C.byref(n)) < 0
    assert lib.srmi_layer_norm_fwd(C.byref(d), big, None, None, big, None, None, None) < 0
    assert lib.srmi_layer_norm_bwd(C.byref(d), big, None, big, big, big, big, big, big, big, big, None) < 0


def test_norm_argument_refusals():
    lib, n = L.load(), C.c_size_t(0)
    d = L.NormDesc(4, 8, L.F32, L.F32, 1e-5, 8, 8)
    big = 1 << 40
    assert lib.srmi_layer_norm_fwd(None, big, None, None, big, None, None, None) == -1
    assert lib.srmi_layer_norm_fwd(C.byref(d), None, None, None, big, None, None, None) == -1
    assert lib.srmi_layer_norm_fwd(C.byref(d), big, None, None, None, None, None, None) == -1
    assert lib.srmi_layer_norm_fwd(C.byref(d), big, None, None, big, big, None, None) == -1              # mean without rstd
    assert lib.srmi_layer_norm_fwd(C.byref(d), big + 1, None, None, big, None, None, None) == -1
    assert lib.srmi_layer_norm_bwd(C.byref(d), big, None, big, big, None, big, None, None, None, 0, None) == -1
    L.check(lib.srmi_layer_norm_workspace_bytes(C.byref(d), C.byref(n)))
    assert lib.srmi_layer_norm_bwd(C.byref(d), big, None, big, big, big, None, big, None, big, n.value - 1, None) == -1
    assert lib.srmi_layer_norm_bwd(C.byref(d), big, None, big, big, big, None, None, None, None, 0, None) == 0     # nothing wanted


def test_dropout_argument_refusals():
    lib, big = L.load(), 1 << 40
    for p in (-0.1, 1.1, float("nan")):
        assert lib.srmi_dropout(big, None, big, 8, L.F32, p, 0, 0, None, None) == -1
    assert lib.srmi_dropout(big, None, big, 8, 7, 0.5, 0, 0, None, None) == -1
    assert lib.srmi_dropout(None, None, big, 8, L.F32, 0.5, 0, 0, None, None) == -1
    assert lib.srmi_dropout(big, None, None, 8, L.F32, 0.5, 0, 0, None, None) == -1
    assert lib.srmi_dropout(big + 1, None, big, 8, L.BF16, 0.5, 0, 0, None, None) == -1
    assert lib.srmi_dropout(big, None, big, 8, L.F32, 0.5, 0, 0, big + 4, None) == -1
    assert lib.srmi_dropout(None, None, None, 0, L.F32, 0.5, 0, 0, None, None) == 0


def test_strided_rows_finds_uniform_strides():
    buf = torch.arange(2 * 3 * 40.).reshape(2, 3, 40)
    t, ld = rows._strided_rows(buf[..., 5:13])
    assert t.data_ptr() == buf[..., 5:13].data_ptr() and ld == 40
    t, ld = rows._strided_rows(buf[:, 1:2, 5:13])
    assert ld == 120 and t.data_ptr() == buf[:, 1:2, 5:13].data_ptr()
    for bad in (buf[:, :2, 5:13], buf.transpose(1, 2), buf[0, :1].expand(4, 40), buf[..., :1].expand(2, 3, 8), buf[0].t()):
        t, ld = rows._strided_rows(bad)
        assert t.is_contiguous() and ld == bad.shape[-1] and torch.equal(t, bad)
    one, ld = rows._strided_rows(buf[:1, :1, 5:13])
    assert ld == 8
    maps = torch.randn(2, 6, 4, 5).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    t, ld = rows._strided_rows(maps)
    assert t is maps and ld == 6


def _calls(x, v, w):
    """every operator with `x` as each of its operands (x [8, 8], v [8], w [8, 8] plain)"""
    return [lambda: rows.linear(x, w), lambda: rows.linear(w, x), lambda: rows.linear(w, w, residual=x), lambda: rows.linear(w, w, x[0]),
            lambda: rows.layer_norm(x), lambda: rows.layer_norm(w, x[0]), lambda: rows.layer_norm(w, v, x[0]),
            lambda: rows.dropout(x, 0.5, 1), lambda: rows.dropout(w, 0.5, 1, residual=x)]


def test_tangents_are_refused():
    # an output without a tangent would pass for a constant
    import torch.autograd.forward_ad as fwAD
    v, w = torch.randn(8), torch.randn(8, 8)
    with fwAD.dual_level():
        x = fwAD.make_dual(torch.randn(8, 8), torch.randn(8, 8))
        for call in _calls(x, v, w):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        with fwAD._set_fwd_grad_enabled(False):                              # nothing to lose
            for call in _calls(x, v, w):
                with pytest.raises(RuntimeError, match="no CPU fallback"):
                    call()


def test_recorders_and_wrapper_tensors_are_refused():
    # a replay would return the memory that the recorded call allocated, unwritten
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, v, w = torch.randn(8, 8), torch.randn(8), torch.randn(8, 8)
    for k in range(9):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(lambda t: _calls(t, v, w)[k](), (x,))
        for mode in ("real", "fake"):
            with pytest.raises(NotImplementedError, match="traced"):
                make_fx(lambda t: _calls(t, v, w)[k](), tracing_mode=mode)(x)
        with FakeTensorMode() as fake:
            t = fake.from_tensor(x)
            with pytest.raises(NotImplementedError, match="traced"):
                _calls(t, v, w)[k]()
        with pytest.raises(NotImplementedError, match="own dispatch"):
            _calls(t, v, w)[k]()
        with pytest.raises(RuntimeError, match="no CPU fallback"):          # as before outside
            _calls(x, v, w)[k]()


def test_dropout_seeds_and_state():
    assert rows.Dropout(0.5).seed is None and rows.Dropout(0.5).state_dict() == {}
    for bad in (-1, 1 << 64):
        with pytest.raises(ValueError, match="seed"):
            rows.Dropout(0.5, seed=bad)
    with pytest.raises(ValueError, match="offset goes with a seed"):
        rows.Dropout(0.5)(torch.randn(3), offset=1)
    net = nn.Sequential(rows.Linear(2, 2), rows.Dropout(0.5, seed=3), rows.Dropout(0.5))
    net[1].calls = (1 << 40) + 5
    state = net.state_dict()
    assert list(state) == ["0.weight", "0.bias", "1.calls"]
    other = nn.Sequential(rows.Linear(2, 2), rows.Dropout(0.5, seed=3), rows.Dropout(0.5))
    other.load_state_dict(state)
    assert other[1].calls == (1 << 40) + 5
    del state["1.calls"]                                                     # a state from before the count was kept
    other.load_state_dict(state)
    assert other[1].calls == (1 << 40) + 5
    state["2.calls"] = torch.tensor(4)                                       # a module without a seed has no count
    with pytest.raises(RuntimeError, match="2.calls"):
        other.load_state_dict(state)


def test_dropout_draws_follow_the_host_generator():
    a, b = rows.Dropout(0.5), rows.Dropout(0.5)
    torch.manual_seed(7)
    first = [a._draw(None), b._draw(None), a._draw(None)]
    torch.manual_seed(7)
    assert first == [a._draw(None), b._draw(None), a._draw(None)]
    assert all(0 <= v < 1 << 64 for pair in first for v in pair) and len({v for pair in first for v in pair}) == 6


@pytest.mark.parametrize("c", [8, 4096, 9000])
@pytest.mark.parametrize("dt", [L.F32, L.BF16])
def test_norm_backward_of_no_rows_is_nothing_to_do(dt, c):
    # dx of no rows: nothing is launched, so this passes without a GPU
    lib, big = L.load(), 1 << 40
    d = L.NormDesc(0, c, dt, dt, 1e-5, c, c)
    assert lib.srmi_layer_norm_bwd(C.byref(d), big, big, big, big, big, big, None, None, None, 0, None) == 0, lib.srmi_last_error()
    assert lib.srmi_layer_norm_bwd(C.byref(d), None, None, None, None, None, big, None, None, None, 0, None) == 0, lib.srmi_last_error()


# ---- how far an f32 product may be off in the root mean square --------------------------------------------------------------
def f32_product_rms(K, sigma, out_rms):
    """root mean square error of a sum of K random products (root mean square `sigma` each) in f32, u = 2^-24.  Added one after the other,
    step k rounds a partial sum of sigma sqrt(k) by at most u of it, evenly: u sigma sqrt(k / 3); the squares add up to
    u^2 sigma^2 K (K + 1) / 6.  Then one rounding of the result.  Sums in blocks or splits stay below."""
    u = 2.0 ** -24
    return u * (sigma * (K * (K + 1) / 6) ** 0.5 + out_rms / 3 ** 0.5)


def _planes(t):
    hi = (t.view(torch.int32) & -65536).view(torch.float32)
    mid = (t - hi).bfloat16().float()
    return hi, mid, (t - hi - mid).bfloat16().float()


@pytest.mark.parametrize("K", [96, 264, 300, 1090, 2100, 2950])
def test_f32_bound_sees_a_missing_plane(K):
    # the kernels multiply f32 as three bf16 planes, six products.  Without the low plane (the three largest products, summed exactly) the
    # error is over the bound at every K the kernels are checked at; with it, and f32 sums of 32 products at a time, under it.
    gen = torch.Generator().manual_seed(K)
    a, b = torch.randn(96, K, generator=gen), torch.randn(160, K, generator=gen)
    want = a.double() @ b.double().t()
    bound = f32_product_rms(K, float(a.double().square().mean().sqrt() * b.double().square().mean().sqrt()), float(want.square().mean().sqrt()))
    pa, pb = _planes(a), _planes(b)

    def total(pairs, exact):
        out = torch.zeros(96, 160, dtype=torch.float64 if exact else torch.float32)
        for k in range(0, K, 32):
            for i, j in pairs:
                part = pa[i][:, k:k + 32].double() @ pb[j][:, k:k + 32].double().t()
                out = out + (part if exact else part.float())
        return float((out.double() - want).square().mean().sqrt())

    assert total([(0, 0), (0, 1), (1, 0)], True) > 1.5 * bound
    assert total([(0, 0), (0, 1), (1, 0), (0, 2), (2, 0), (1, 1)], False) <= bound
