"""The MoE experts layer of a decode batch, in two launches.

Stands beside ``VllmFusedExperts`` (same ``forward`` arguments) for at most 64
tokens: one launch for the gate and up products with SiLU*Mul, one for the down
product with the routed sum.  The activations are not quantized, so its
results are nearer to the exact ones than those of the FP8 x FP8 chain, and
the weights may also be MXFP4.  No other layer takes MXFP4 experts: more tokens
go through them 64 at a time, and each call reads the named experts' weights.

With many rows an expert (tokens that name it) the sorted-token layer is the
faster one for FP8 weights: up to ten on average this one takes at most 1.05 of
its time, at sixteen up to 1.5.  The kernels' sizes go by T * top_k / E rows, as for
uniform routing with every id inside [0, E); other routings give the same results
in more time than they need.  For inference, as the rest of the package: the
output carries no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _ops
from ._ops import FP8, GROUP, MX_GROUP


class FewTokenExperts(nn.Module):
    """``forward(hidden_states, w13, w2, topk_weights, topk_ids, num_experts,
    w13_scale, w2_scale, block_shape)``: bf16 or fp16 [T, H] hidden states, T <=
    64 (``MAX_TOKENS``); routing fp32 weights and int32 or int64 ids [T, top_k].

    ``block_shape`` [128, 128]: fp8 w13 [E, 2I, H] (gate rows, then up rows) and
    w2 [E, H, I] with fp32 block scales, used as given.  [1, 32]: MXFP4 codes
    [E, 2I, H/2] and [E, H, I/2] with scales [E, 2I, H/32] and [E, H, I/32].

    Returns [T, H] in the hidden states' dtype.  Ids outside [0, E) (experts of
    other ranks, padding tokens) count for nothing."""

    MAX_TOKENS = _ops.FEW_TOKENS

    def forward(self, hidden_states: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor,
                topk_ids: torch.Tensor, num_experts: int, w13_scale: torch.Tensor, w2_scale: torch.Tensor,
                block_shape: list[int]) -> torch.Tensor:
        expected = [GROUP, GROUP] if w13.dtype is FP8 else [1, MX_GROUP]
        if list(block_shape) != expected:
            raise ValueError(f"FewTokenExperts: block_shape must be {expected} for {w13.dtype} weights, got {block_shape}")
        if num_experts != w13.shape[0]:
            raise ValueError(f"FewTokenExperts: num_experts={num_experts}, but w13 holds {w13.shape[0]}")
        if _ops._host is not None and not torch.compiler.is_compiling():
            out = _ops._host.few_experts(hidden_states, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids)
            if out is not None:
                return out
        out = torch.empty(hidden_states.shape, dtype=hidden_states.dtype, device=hidden_states.device)
        args = (hidden_states, w13, w13_scale, w2, w2_scale, topk_weights.contiguous(), topk_ids.contiguous(), out)
        if torch.compiler.is_compiling():
            torch.ops.kb_nano_fp8_moe.few_token_experts(*args)
        else:
            _ops.few_token_experts(*args)
        return out
