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
kept between calls (workspaces come from torch's allocator, call by call), so graphs and streams share nothing.  Capturing a
differentiable call whose leaves an eager autograd graph of the default stream still refers to is refused (autograd would end the process
in the captured backward pass): delete that graph first, or run warm-ups on a side stream.

Gradients are first derivatives in reverse mode; a tensor with a tangent of forward-mode AD raises.  So does a call that is being traced
or exported, and a tensor subclass with its own dispatch (DTensor, FakeTensor).

Reference call sites these stand next to: ``nn.Linear`` + LeakyReLU (P/srgan_model.py:57-60), ``nn.BatchNorm2d`` (P/ops.py:24-26).
The checks, tensors and autograd nodes are in csrc/rows_torch.cpp.  No fallback: CPU tensors raise; no ATen arithmetic.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib as L
from . import functional as Fn


def _act_of(act):
    """activation module -> (code, parameter) of the row operators"""
    if act is None:
        return L.ACT_NONE, 0.0
    if isinstance(act, nn.GELU):
        return (L.ACT_GELU_TANH if act.approximate == "tanh" else L.ACT_GELU), 0.0
    if isinstance(act, nn.SiLU):
        return L.ACT_SILU, 0.0
    if isinstance(act, (nn.PReLU, Fn.AddReLU)):
        raise NotImplementedError(f"srmi.rows: {type(act).__name__} is an epilogue of the convolutions (autograd.linear), not of rows.linear")
    code, param, _, _ = Fn.act_of(act)
    return code, param


def _tensor(t, what, optional=False):
    if not (isinstance(t, torch.Tensor) or (optional and t is None)):
        raise TypeError(f"srmi.rows: {what} must be a tensor, got {type(t).__name__}")


def _strided_rows(t):
    """(tensor, row stride) of `t` seen as [rows, t.shape[-1]]: in place if the leading axes walk with one stride, else a copy."""
    return L.load_rows().strided_rows(t)


def linear(x, weight, bias=None, act=None, residual=None):
    """``act(x @ weight.T + bias) + residual`` in one pass.  x [..., K], weight [N, K], bias [N], residual [..., N]; ``act``: None, or
    an nn.ReLU / LeakyReLU / Tanh / Sigmoid / GELU (either form) / SiLU module.  All tensors share x's dtype (float32: the products
    have float32's accuracy, operands below 2^-110 being taken to the nearest 2^-133; bfloat16: bf16 operands, f32 sums).

    Training in bfloat16 rounds ``dy * act'(z)`` to bfloat16 once, as the products' operand (the bias gradient sums it before that
    rounding); the pre-activation is kept as an IEEE half.  A float32 infinity in x or weight may come out as NaN."""
    _tensor(x, "x")
    _tensor(weight, "weight")
    _tensor(bias, "bias", True)
    _tensor(residual, "residual", True)
    code, param = _act_of(act)
    return L.load_rows().linear(x, weight, bias, residual, code, param)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last axis: ``(x - mean) / sqrt(var + eps) * weight + bias``.  weight, bias [C]: None, x's dtype, or float32
    parameters next to bfloat16 rows (both the same)."""
    _tensor(x, "x")
    _tensor(weight, "weight", True)
    _tensor(bias, "bias", True)
    return L.load_rows().layer_norm(x, weight, bias, float(eps))


def dropout(x, p, seed, offset=0, residual=None):
    """``residual + dropout(x)``: every element of x is dropped with probability ``p`` or scaled by ``1 / (1 - p)``.

    The mask is a function of (seed, offset, index of the element in row-major order) and is never stored; the backward pass
    computes it again.  ``seed`` and ``offset`` are integers in [0, 2^64): use one seed per site (and rank) and a new offset per step.
    ``seed`` may instead be an int64 CUDA tensor ``[seed, offset]`` that the kernel reads, so that a captured graph draws a new mask
    at every replay; write it only before a forward or after that forward's backward."""
    _tensor(x, "x")
    _tensor(residual, "residual", True)
    rng = None
    if isinstance(seed, torch.Tensor):
        if offset != 0:
            raise ValueError("srmi.rows.dropout: a device tensor holds seed and offset, pass no other offset")
        rng, seed = seed, 0
    else:
        for v, what in ((seed, "seed"), (offset, "offset")):
            if isinstance(v, bool) or not isinstance(v, int) or not 0 <= v < 1 << 64:
                raise ValueError(f"srmi.rows.dropout: {what} must be an integer in [0, 2^64), got {v!r}")
    return L.load_rows().dropout(x, residual, float(p), seed, offset, rng)


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
    """Dropout with a residual add; identity (plus the residual) in eval mode.

    ``seed=None``: every call in training draws a seed and an offset from torch's host generator.  ``torch.manual_seed`` repeats a run, modules
    differ, and activation checkpointing (`torch.utils.checkpoint` restores that generator) recomputes with the forward's mask.
    Seed the generator differently on every data-parallel rank.

    With an integer ``seed`` nothing else decides: call number k of this module in training draws with offset k (``calls``, kept in the
    state_dict so that a resumed run goes on).  Give every module - and every rank - its own.  A call that is recomputed inside a backward
    pass would count again and draw another mask: it raises, pass ``offset`` there, a number that names the call (a step), instead of
    the count.

    While a HIP graph is being captured any host-side number would repeat one mask at every replay: pass ``rng``, the device tensor
    of `dropout`."""

    def __init__(self, p=0.5, seed=None):
        super().__init__()
        if not 0.0 <= float(p) <= 1.0:
            raise ValueError(f"srmi.rows.Dropout: p must be in [0, 1], got {p}")
        if seed is not None and not 0 <= int(seed) < 1 << 64:
            raise ValueError(f"srmi.rows.Dropout: seed must be None or an integer in [0, 2^64), got {seed}")
        self.p, self.seed, self.calls = float(p), None if seed is None else int(seed), 0

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        if self.seed is not None:
            destination[prefix + "calls"] = torch.tensor(self.calls, dtype=torch.int64, device="cpu")

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        key = prefix + "calls"
        if self.seed is not None and key in state_dict:
            self.calls = int(state_dict[key])
            if key in unexpected_keys:
                unexpected_keys.remove(key)

    @torch.compiler.disable
    def _draw(self, offset):
        """(seed, offset) of this call"""
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("srmi.rows.Dropout: pass rng=[seed, offset] (int64 device tensor) inside a graph capture")
        if self.seed is None:
            if offset is not None:
                raise ValueError("srmi.rows.Dropout: offset goes with a seed, this module has none")
            return [v % (1 << 64) for v in torch.randint(-(1 << 63), (1 << 63) - 1, (2,), dtype=torch.int64, device="cpu").tolist()]
        if offset is not None:
            return self.seed, offset
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("srmi.rows.Dropout: a module with a seed counts its calls, and this one is recomputed inside a backward pass "
                               "(activation checkpointing): pass offset, or leave seed=None")
        self.calls += 1
        return self.seed, self.calls

    def forward(self, x, residual=None, rng=None, offset=None):
        if not self.training:
            return x if residual is None else dropout(x, 0.0, 0, residual=residual)
        if rng is not None:
            return dropout(x, self.p, rng, 0 if offset is None else offset, residual=residual)
        return dropout(x, self.p, *self._draw(offset), residual=residual)
