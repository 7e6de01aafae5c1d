"""Operators on rows of features: linear layers with a fused epilogue, layer norm and counter-based dropout, with backward.

A row is one token, or one pixel of a channels-last map: tensors are ``[..., C]`` and every leading axis counts rows.  What the
convolutions of this package hand out (logical NCHW, channels_last storage) enters without a copy::

    rows_ = feat.permute(0, 2, 3, 1)                          # [N, H, W, C] view of a channels_last map
    h = rows.linear(rows.layer_norm(rows_, g, b), w1, b1, act=nn.GELU())
    h = rows.linear(h, w2, b2)
    out = rows.dropout(h, 0.1, seed, step, residual=rows_).permute(0, 3, 1, 2)

Storage is float32 or bfloat16 (one type per call); sums, statistics and activations are float32.  Rows may be strided (a
channel slice of a wider buffer is read in place); anything whose last axis is not dense is copied first.  Outputs are dense.
Results do not depend on timing: no atomics, the same call gives the same bits.  Calls may be captured into a HIP graph; nothing is
kept between calls (workspaces come from torch's allocator, call by call), so graphs and streams share nothing.  As with any torch
operator, capture a backward pass with leaves that no eager graph still alive has used (``torch.autograd.grad`` avoids the
accumulation nodes altogether).

Reference call sites these stand next to: ``nn.Linear`` + LeakyReLU (P/srgan_model.py:57-60), ``nn.BatchNorm2d`` (P/ops.py:24-26).
No fallback: CPU tensors raise; no ATen arithmetic.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import functional as Fn

_NULL = contextlib.nullcontext()


def _act_of(act):
    """activation module -> (code, parameter) of the row operators"""
    if isinstance(act, nn.GELU):
        return (L.ACT_GELU_TANH if act.approximate == "tanh" else L.ACT_GELU), 0.0
    if isinstance(act, nn.SiLU):
        return L.ACT_SILU, 0.0
    if isinstance(act, (nn.PReLU, Fn.AddReLU)):
        raise NotImplementedError(f"srmi.rows: {type(act).__name__} is an epilogue of the convolutions (autograd.linear), not of rows.linear")
    code, param, _, _ = Fn.act_of(act)
    return code, param


def _check(t, what, dtype, device, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"srmi.rows: {what} must be a tensor, got {type(t).__name__}")
    Fn.require_cuda(t, what)
    if t.dtype != dtype:
        raise TypeError(f"srmi.rows: {what} is {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"srmi.rows: {what} is on {t.device}, x on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"srmi.rows: {what} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _check_x(x):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"srmi.rows: x must be a tensor, got {type(x).__name__}")
    Fn.require_cuda(x)
    if x.dim() < 1:
        raise ValueError("srmi.rows: x needs at least one axis")
    return Fn.dtype_code(x.dtype)


def _on(device):
    """the launches go to the tensors' device, whichever is current"""
    return _NULL if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _strided_rows(t):
    """(tensor, row stride) of `t` seen as [rows, t.shape[-1]]: in place if the leading axes walk with one stride, else a copy."""
    c = t.shape[-1]
    if t.is_contiguous():
        return t, c
    if t.stride(-1) == 1 or c <= 1:
        ld, n = None, 1                        # stride of the innermost leading axis longer than one, rows below it
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if ld is None:
                ld = stride
            elif stride != ld * n:
                ld = -1
                break
            n *= size
        if ld is None:
            ld = c
        if ld >= max(c, 1):
            return t, ld
    return t.contiguous(), c


def _ptr(t):
    return t.data_ptr() if t is not None else None


_DESCS = {}


def _linear_desc(*key):
    """(descriptor, forward / backward workspace bytes) of one shape, kept: building them costs more than a small launch"""
    hit = _DESCS.get(key)
    if hit is None:
        d = L.LinearDesc(*key)
        sizes = []
        for which in (L.PASS_FWD, L.PASS_BWD):
            n = C.c_size_t(0)
            L.check(L.load().srmi_linear_workspace_bytes(C.byref(d), which, C.byref(n)))
            sizes.append(n.value)
        if len(_DESCS) > 4096:
            _DESCS.clear()
        hit = _DESCS[key] = (d, C.byref(d), sizes[0], sizes[1])
    return hit


def _align(*tensors):
    """what the library may assume of the pointers: 16 bytes, or just their element"""
    bits = 0
    for t in tensors:
        if t is not None:
            bits |= t.data_ptr()
    return 0 if bits & 15 else 16


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear_fwd(x, weight, bias, residual, act, param, want_z):
    N, K = weight.shape
    out_shape = x.shape[:-1] + (N,)
    xr, ldx = _strided_rows(x)
    wr, ldw = _strided_rows(weight)
    rr, ldr = (None, 0) if residual is None else _strided_rows(residual)
    M = out_shape.numel() // N if N else 0
    y = torch.empty(out_shape, dtype=x.dtype, device=x.device)
    z = torch.empty((M, N), dtype=x.dtype, device=x.device) if want_z else None
    if M and N:
        b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        with _on(x.device):
            _, ref, ws_fwd, _ = _linear_desc(M, N, K, Fn.dtype_code(x.dtype), act, param, _align(xr, wr), ldx, ldw, ldr, 0)
            ws = _workspace(ws_fwd, x.device)
            L.check(L.load().srmi_linear_fwd(ref, xr.data_ptr(), wr.data_ptr(), _ptr(b), _ptr(rr), y.data_ptr(), _ptr(z), _ptr(ws),
                                             ws_fwd, Fn.stream_ptr(x.device)))
    return y, z, xr, wr


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, param):
        need = ctx.needs_input_grad
        slope = act != L.ACT_NONE and any(need[:3])
        # ReLU and LeakyReLU keep the sign of z: without a residual on top y itself is enough for the backward pass
        by_sign = residual is None and (act == L.ACT_RELU or (act == L.ACT_LRELU and param > 0.0))
        y, z, xr, wr = _linear_fwd(x, weight, bias, residual, act, param, slope and not by_sign)
        ctx.save_for_backward(xr if need[1] else None, wr if need[0] else None, (y if by_sign else z) if slope else None)
        ctx.cfg = act, param, x.shape, weight.shape, bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, saved = ctx.saved_tensors
        act, param, xshape, (N, K), has_bias = ctx.cfg
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dev, dt = dy.device, dy.dtype
            dyr, lddy = _strided_rows(dy)
            ldx = _strided_rows(x)[1] if x is not None else K
            ldw = _strided_rows(w)[1] if w is not None else K
            M = xshape.numel() // K if K else dy.numel() // max(N, 1)
            if need[0]:
                dx = torch.empty(xshape, dtype=dt, device=dev)
            if need[1]:
                dw = torch.empty((N, K), dtype=dt, device=dev)
            if need[2] and has_bias:
                db = torch.empty((N,), dtype=dt, device=dev)
            with _on(dev):
                _, ref, _, ws_bwd = _linear_desc(M, N, K, Fn.dtype_code(dt), act, param, _align(x, w, dyr), ldx, ldw, 0, lddy)
                ws = _workspace(ws_bwd, dev)
                L.check(L.load().srmi_linear_bwd(ref, _ptr(x), _ptr(w), _ptr(saved), dyr.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
                                                 ws_bwd, Fn.stream_ptr(dev)))
        return dx, dw, db, dy if need[3] else None, None, None


def linear(x, weight, bias=None, act=None, residual=None):
    """``act(x @ weight.T + bias) + residual`` in one pass.  x [..., K], weight [N, K], bias [N], residual [..., N]; ``act``: None, or
    an nn.ReLU / LeakyReLU / Tanh / Sigmoid / GELU (either form) / SiLU module.  All tensors share x's dtype (float32: the products
    have float32's accuracy; bfloat16: bf16 operands, f32 sums).

    Training in bfloat16 keeps the pre-activation and forms ``dy * act'(z)`` in bfloat16, one rounding each (the bias gradient
    sums the products before that rounding)."""
    _check_x(x)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("srmi.rows.linear: weight must be [out_features, in_features]")
    _check(weight, "weight", x.dtype, x.device)
    N, K = weight.shape
    if x.shape[-1] != K:
        raise ValueError(f"srmi.rows.linear: x has {x.shape[-1]} features, weight {tuple(weight.shape)}")
    if bias is not None:
        _check(bias, "bias", x.dtype, x.device, (N,))
    if residual is not None:
        _check(residual, "residual", x.dtype, x.device, x.shape[:-1] + (N,))
    code, param = _act_of(act)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _LinearFn.apply(x, weight, bias, residual, code, param)
    return _linear_fwd(x, weight, bias, residual, code, param, False)[0]


def _norm_desc(rows, c, dtype, param_dtype, eps, ldx, lddy):
    return L.NormDesc(rows, c, dtype, param_dtype, eps, ldx, lddy)


def _norm_fwd(x, weight, bias, eps, keep):
    c = x.shape[-1]
    rows = x.numel() // c
    xr, ldx = _strided_rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    p = weight if weight is not None else bias
    pd = Fn.dtype_code(p.dtype) if p is not None else L.F32
    if rows:
        w = weight if weight is None or weight.is_contiguous() else weight.contiguous()
        b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        with _on(x.device):
            d = _norm_desc(rows, c, Fn.dtype_code(x.dtype), pd, eps, ldx, 0)
            base = _ptr(stats)
            L.check(L.load().srmi_layer_norm_fwd(C.byref(d), xr.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(), base,
                                                 base + 4 * rows if keep else None, Fn.stream_ptr(x.device)))
    return y, stats, xr, ldx


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats, xr, ldx = _norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(xr, weight, stats)
        p = weight if weight is not None else bias
        ctx.cfg = eps, x.shape, ldx, p.dtype if p is not None else torch.float32
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xr, weight, stats = ctx.saved_tensors
        eps, shape, ldx, pdt = ctx.cfg
        need = ctx.needs_input_grad
        c, dev = shape[-1], dy.device
        rows = stats.shape[1]
        dyr, lddy = _strided_rows(dy)
        dx = torch.empty(shape, dtype=dy.dtype, device=dev) if need[0] else None
        dw = torch.empty((c,), dtype=pdt, device=dev) if need[1] else None
        db = torch.empty((c,), dtype=pdt, device=dev) if need[2] else None
        if weight is not None and not weight.is_contiguous():
            weight = weight.contiguous()
        lib = L.load()
        with _on(dev):
            d = _norm_desc(rows, c, Fn.dtype_code(dy.dtype), Fn.dtype_code(pdt), eps, ldx, lddy)
            nbytes = 0
            if dw is not None or db is not None:
                n = C.c_size_t(0)
                L.check(lib.srmi_layer_norm_workspace_bytes(C.byref(d), C.byref(n)))
                nbytes = n.value
            ws = _workspace(nbytes, dev)
            base = stats.data_ptr()
            L.check(lib.srmi_layer_norm_bwd(C.byref(d), xr.data_ptr(), _ptr(weight), base, base + 4 * rows, dyr.data_ptr(), _ptr(dx), _ptr(dw),
                                            _ptr(db), _ptr(ws), nbytes, Fn.stream_ptr(dev)))
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last axis: ``(x - mean) / sqrt(var + eps) * weight + bias``.  weight, bias [C]: None, x's dtype, or float32
    parameters next to bfloat16 rows (both the same)."""
    _check_x(x)
    c = x.shape[-1]
    if c == 0:
        raise ValueError("srmi.rows.layer_norm: the last axis is empty")
    if not eps >= 0.0:
        raise ValueError("srmi.rows.layer_norm: eps must be >= 0")
    pdt = None
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if pdt is None:
            pdt = t.dtype if isinstance(t, torch.Tensor) and t.dtype == torch.float32 else x.dtype
        _check(t, what, pdt, x.device, (c,))
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _norm_fwd(x, weight, bias, float(eps), False)[0]


def _dropout_run(x, residual, p, seed, offset, rng):
    x = x.contiguous()
    r = residual.contiguous() if residual is not None else None
    y = torch.empty_like(x)
    if x.numel():
        with _on(x.device):
            L.check(L.load().srmi_dropout(x.data_ptr(), _ptr(r), y.data_ptr(), x.numel(), Fn.dtype_code(x.dtype), p, seed, offset, _ptr(rng),
                                          Fn.stream_ptr(x.device)))
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, rng):
        ctx.save_for_backward(rng)              # an in-place write between the passes would change the mask: torch reports it
        ctx.cfg = p, seed, offset
        return _dropout_run(x, residual, p, seed, offset, rng)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = _dropout_run(dy, None, *ctx.cfg, rng) if need[0] else None
        return dx, dy if need[1] else None, None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """``residual + dropout(x)``: every element of x is dropped with probability ``p`` or scaled by ``1 / (1 - p)``.

    The mask is a function of (seed, offset, index of the element in row-major order) and is never stored; the backward pass
    computes it again.  ``seed`` and ``offset`` are integers in [0, 2^64): use one seed per site (and rank) and a new offset per step.
    ``seed`` may instead be an int64 CUDA tensor ``[seed, offset]`` that the kernel reads, so that a captured graph draws a new mask
    at every replay; write it only before a forward or after that forward's backward."""
    _check_x(x)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"srmi.rows.dropout: p must be in [0, 1], got {p}")
    rng = None
    if isinstance(seed, torch.Tensor):
        if offset != 0:
            raise ValueError("srmi.rows.dropout: a device tensor holds seed and offset, pass no other offset")
        _check(seed, "seed", torch.int64, x.device, (2,))
        if not seed.is_contiguous():
            raise ValueError("srmi.rows.dropout: the [seed, offset] tensor must be contiguous")
        rng, seed = seed, 0
    else:
        for v, what in ((seed, "seed"), (offset, "offset")):
            if isinstance(v, bool) or not isinstance(v, int) or not 0 <= v < 1 << 64:
                raise ValueError(f"srmi.rows.dropout: {what} must be an integer in [0, 2^64), got {v!r}")
    if residual is not None:
        _check(residual, "residual", x.dtype, x.device, x.shape)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutFn.apply(x, residual, p, seed, offset, rng)
    return _dropout_run(x, residual, p, seed, offset, rng)


class Linear(nn.Linear):
    """`nn.Linear` (same parameters and state_dict keys) with the activation and the residual add in its epilogue."""

    def __init__(self, in_features, out_features, bias=True, act=None, device=None, dtype=None):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        _act_of(act)
        self.act = act

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, act=self.act, residual=residual)


class LayerNorm(nn.LayerNorm):
    """`nn.LayerNorm` over the last axis (same parameters and state_dict keys)."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError("srmi.rows.LayerNorm: one normalised axis, the last")

    def forward(self, x):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"srmi.rows.LayerNorm: x has shape {tuple(x.shape)}, normalised are {self.normalized_shape}")
        return layer_norm(x, self.weight, self.bias, self.eps)


class Dropout(nn.Module):
    """Dropout with a residual add; call number k of this module in training draws with offset k under its seed (``calls``, reset or
    restore it to repeat a run).  Give every module - and every data-parallel rank - its own seed.  Identity (plus the residual)
    in eval mode.  While a graph is being captured a host-side count would repeat one mask at every replay: pass ``rng``, the device
    tensor of `dropout`, there."""

    def __init__(self, p=0.5, seed=0):
        super().__init__()
        if not 0.0 <= float(p) <= 1.0:
            raise ValueError(f"srmi.rows.Dropout: p must be in [0, 1], got {p}")
        self.p, self.seed, self.calls = float(p), int(seed), 0

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"

    def forward(self, x, residual=None, rng=None):
        if not self.training:
            return x if residual is None else dropout(x, 0.0, 0, residual=residual)
        if rng is not None:
            return dropout(x, self.p, rng, residual=residual)
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("srmi.rows.Dropout: pass rng=[seed, offset] (int64 device tensor) inside a graph capture")
        self.calls += 1
        return dropout(x, self.p, self.seed, self.calls, residual=residual)
