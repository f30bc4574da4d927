"""cute_triadic_gdn_b200: hand-written sm_100a CUDA kernels for Triadic Gated DeltaNet behind the reference's Python API.

    chunk_gdn_joint       Triadic GDN with autograd, as a plain autograd call
    gdn_joint_call        the same behind torch.library custom ops (one node under torch.compile)
    conv_split_act_call   causal depthwise convolution (width 4) with SiLU on the leading channels only

Same names, signatures, shapes and dtypes as cute_triadic_gdn/__init__.py:7-11 of the reference.

Beyond the reference's surface:

    conv_split_norm_call            the convolution with the layer glue fused in: x -> (q, k, v, k2, q2) as the core
                                    takes them (SiLU / softplus, l2 norms), differentiable
    gdn_joint_decode                one token per sequence on a resident state (continues what
                                    chunk_gdn_joint(..., output_final_state=True) hands out)
    chunk_gdn_joint_segment         one segment of longer sequences: state in / state out, differentiable through both
    context_parallel_joint          sequences split along the token axis over the ranks of a process group (states and
                                    their gradients travel point to point, head groups as a wavefront)
    gated_scan_call                 per-channel gated linear recurrence h[t] = exp(g[t]) h[t-1] + x[t]: dense or packed rows, state in and
                                    out, differentiable through both
    gated_scan_decode               its decode step: one token per sequence on a resident state
    residual_norm_call              before a block: residual stream + scale * x and its norm in one pass
    gated_norm_call                 after a block: norm, gate and, where asked for, the scaled sum into the residual stream
    HostPipeline / gdn_joint_host   inputs and results in pinned host memory; uploads, kernels and downloads of
                                    successive batch slices overlap on three streams (host_pipeline.py)
"""
from .block_norm import gated_norm_call, residual_norm_call
from .conv_split_act import conv_split_act_call, conv_split_norm_call
from .context_parallel import context_parallel_joint
from .gated_scan import gated_scan_call, gated_scan_decode
from .gdn_joint import chunk_gdn_joint, chunk_gdn_joint_segment, gdn_joint_decode
from .host_pipeline import HostPipeline, gdn_joint_host
from .joint_torch_ops import gdn_joint_call

__all__ = ["chunk_gdn_joint", "gdn_joint_call", "conv_split_act_call", "conv_split_norm_call", "gdn_joint_decode", "chunk_gdn_joint_segment",
           "context_parallel_joint", "gated_scan_call", "gated_scan_decode", "residual_norm_call", "gated_norm_call", "HostPipeline",
           "gdn_joint_host"]
__version__ = "0.1.0"
