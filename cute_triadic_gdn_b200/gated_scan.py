"""Gated linear recurrence per channel: `gated_scan_call` and its decode step `gated_scan_decode`.

    h[t] = exp(g[t]) h[t-1] + x[t]

The recurrence of the layers that alternate with the matrix-state core in a hybrid stack: a vector state instead of E x 128 x 128 per head,
gates as logs of decays like the core's.  No counterpart in the reference.  The device work is csrc/tgdn_scan.cu; checks, autograd and
launches are in csrc/tgdn_torch_block.cpp.
"""
from __future__ import annotations

import torch

from . import _lib
from .joint_packing import _validate


@torch.library.register_fake("tgdn_b200::gated_scan_map")
def _map_fake(cu_seqlens, tokens):
    return cu_seqlens.new_empty(tokens, dtype=torch.int32), cu_seqlens.new_empty(1, dtype=torch.bool)


@torch.library.register_fake("tgdn_b200::gated_scan_fwd")
def _fwd_fake(x, g, initial_state=None, doc_map=None, documents=0, output_final_state=False, save=False):
    B, T, D = x.shape
    f32 = lambda *shape: x.new_empty(shape, dtype=torch.float32)
    final = f32(B if doc_map is None else documents, D) if output_final_state else f32(0)
    return torch.empty_like(x, memory_format=torch.contiguous_format), final, f32(B * ((T + 127) // 128) * D) if save else f32(0)


@torch.library.register_fake("tgdn_b200::gated_scan_bwd")
def _bwd_fake(x, g, dh, carry, initial_state=None, doc_map=None, documents=0, dfinal=None):
    contiguous = torch.contiguous_format
    dinitial = x.new_empty(0, dtype=torch.float32) if initial_state is None else torch.empty_like(initial_state, memory_format=contiguous)
    return torch.empty_like(x, memory_format=contiguous), torch.empty_like(g, memory_format=contiguous), dinitial


def gated_scan_call(x, g, cu_seqlens=None, *, initial_state=None, output_final_state=False):
    """h (B, T, D) of h[t] = exp(g[t]) h[t-1] + x[t], every channel by itself, states in f32; h has x's type.

    x: (B, T, D) f32, bf16 or f16; g: logs of decays (g <= 0 for a state that forgets; above zero it grows; -inf drops a finite state), f32 or
    of x's type.  exp(g) and the states are f32: a gate above 88.7 is infinite growth, and a state, or a product of decays, below 2^-126 counts
    as zero.  Any strides over batch and tokens are read in place (a slice of a projection, an expanded gate).  `initial_state`: f32
    (sequences, D), zero if not given; with `output_final_state=True` the call returns (h, final_state).  Differentiable in x, g and initial_state, through h and final_state, so
    that sequences can be processed in segments.

    With cu_seqlens the inputs are one packed row (1, T, D) as in `gdn_joint_call`: contiguous int32/int64 CUDA offsets that start at 0, end
    at T and strictly increase; every document starts from its own state (sequences = documents).

    A sequence's results do not depend on what runs beside it in the batch."""
    if not torch.compiler.is_compiling():
        h, final = _lib.host.scan_call(x, g, cu_seqlens, initial_state, bool(output_final_state))
        return (h, final) if output_final_state else h
    doc_map, documents = None, 0
    if cu_seqlens is not None:
        _validate((x,), cu_seqlens)
        documents = cu_seqlens.numel() - 1
        doc_map, valid = torch.ops.tgdn_b200.gated_scan_map(cu_seqlens, x.shape[1])
        torch._assert_async(valid, "cu_seqlens must start at 0, end at T, and strictly increase")
    h, final, _ = torch.ops.tgdn_b200.gated_scan_fwd(x, g, initial_state, doc_map, documents, bool(output_final_state), False)
    return (h, final) if output_final_state else h


def gated_scan_decode(x, g, state):
    """One token per sequence on a resident state: continues what `gated_scan_call(..., output_final_state=True)` hands out.

    x, g: (B, 1, D) or (B, D), types as in `gated_scan_call`; `state`: contiguous f32 (B, D), updated IN PLACE to exp(g) state + x.  Returns
    the new state in x's type and shape.  Forward only."""
    return _lib.host.scan_decode(x, g, state)
