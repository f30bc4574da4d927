"""Norms before and after a block, fused with the residual stream, its scale and the block's gate: `residual_norm_call`, `gated_norm_call`.

What stands around the core in a layer and what the reference leaves to its caller: the residual sum and the norm in front of the projections,
the gated norm of the heads' outputs (and, for norms behind a block, the scaled sum into the stream).  The device work is csrc/tgdn_norm.cu and
csrc/tgdn_gated_norm.cu; checks, autograd and launches are in csrc/tgdn_torch_block.cpp.
"""
from __future__ import annotations

import torch

from . import _lib

_ACTIVATIONS = {"silu": 1, "sigmoid": 2}


def _like(t, dtype=None):
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _rstd(x, save):
    return x.new_empty(x.shape[:-1].numel() if save else 0, dtype=torch.float32)


def _none(x):
    return x.new_empty(0, dtype=torch.float32)


@torch.library.register_fake("tgdn_b200::residual_norm_fwd")
def _residual_fwd_fake(x, residual, weight, scale, scale_value, eps, save=False):
    return _like(x), _like(residual), _rstd(x, save)


@torch.library.register_fake("tgdn_b200::residual_norm_bwd")
def _residual_bwd_fake(stream, x, x_type, dy, dstream, weight, scale, scale_value, rstd, want_weight, want_scale):
    same = scale is None and scale_value == 1.0 and x_type == stream.dtype
    return (_like(stream), _none(stream) if same else _like(stream, x_type), _like(weight) if want_weight else _none(stream),
            _like(scale) if want_scale else _none(stream))


@torch.library.register_fake("tgdn_b200::gated_norm_fwd")
def _gated_fwd_fake(x, gate, weight, residual, scale, scale_value, activation, eps, save=False):
    return _like(x, None if residual is None else residual.dtype), _rstd(x, save)


@torch.library.register_fake("tgdn_b200::gated_norm_bwd")
def _gated_bwd_fake(x, gate, dout, weight, scale, scale_value, activation, rstd, want_weight, want_scale):
    return (_like(x), _none(x) if gate is None else _like(x), _like(weight) if want_weight else _none(x), _like(scale) if want_scale else _none(x))


def _scale(scale):
    """(vector over the channels or None, number)"""
    if torch.is_tensor(scale):
        return scale, 1.0
    return None, 1.0 if scale is None else float(scale)


def residual_norm_call(x, residual, weight=None, scale=None, eps=1e-6):
    """The residual sum and the norm before a block in one pass: returns (y, stream) with

        stream = residual + scale * x,        y = stream * rsqrt(mean(stream^2) + eps) * weight

    over the last axis (at most 16384 channels).  x: (..., N) f32, bf16 or f16, the output of the block before; residual: x's shape, f32 or
    x's type; `stream` has the residual's type (the next call's residual), `y` x's.  The norm is taken of the sum before it is rounded to the
    stream's type; the backward forms it from the stream as stored (with a 16-bit stream, gradients of f32 vectors are as good as its type).  weight: (N), ones if not given; scale: a number or a vector (N), one if not
    given.  Differentiable in all four tensors.  Rows are read in place where their strides allow it."""
    vector, value = _scale(scale)
    if not torch.compiler.is_compiling():
        return _lib.host.residual_norm(x, residual, weight, vector, value, float(eps))
    y, stream, _ = torch.ops.tgdn_b200.residual_norm_fwd(x, residual, weight, vector, value, float(eps))
    return y, stream


def gated_norm_call(x, gate=None, weight=None, residual=None, scale=None, activation="silu", eps=1e-6):
    """The norm after a block with its gate, and where `residual` is given the scaled sum into the stream:

        y = x * rsqrt(mean(x^2) + eps) * weight * act(gate),        returns scale * y  or  residual + scale * y

    over the last axis (at most 16384 channels): heads of 128 as the core returns them, or whole rows.  x: (..., N) f32, bf16 or f16; gate:
    like x (a slice of a projection is read in place) or None for a plain norm; activation: "silu" or "sigmoid"; residual: x's shape, f32 or
    x's type, and then the result's type; weight, scale as in `residual_norm_call`.  Differentiable in all five tensors."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation: one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    vector, value = _scale(scale)
    act = 0 if gate is None else _ACTIVATIONS[activation]
    if not torch.compiler.is_compiling():
        return _lib.host.gated_norm(x, gate, weight, residual, vector, value, act, float(eps))
    return torch.ops.tgdn_b200.gated_norm_fwd(x, gate, weight, residual, vector, value, act, float(eps))[0]
