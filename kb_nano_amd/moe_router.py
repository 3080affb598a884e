"""Routing of tokens to experts: the router's product and the choice of experts.

No counterpart in kb_nano's FP8 path; the modules make what ``FusedExperts``,
``VllmFusedExperts`` and ``FewTokenExperts`` take (``topk_weights``,
``topk_ids``).  For inference, as the rest of the package: outputs carry no
gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _ops


class MoeRouterGemm(nn.Module):
    """``forward(hidden_states, weight) -> logits``: bf16, fp16 or fp32 hidden
    states ``[..., H]`` (H % 8 == 0) times ``weight [E, H]`` (of their type or
    fp32, as checkpoints keep it), fp32 logits ``[..., E]`` from fp32 sums: no
    rounding between the product and the choice of experts.  Infinities give the
    formula's infinities and NaN, whatever the types and the number of tokens."""

    def forward(self, hidden_states: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        if _ops._host is not None and not torch.compiler.is_compiling():
            out = _ops._host.router_gemm(hidden_states, weight)   # the plain case in one native step
            if out is not None:
                return out
        x2 = hidden_states if hidden_states.dim() == 2 else hidden_states.reshape(-1, hidden_states.shape[-1])
        out = torch.empty(x2.shape[0], weight.shape[0], dtype=torch.float32, device=x2.device)
        if torch.compiler.is_compiling():
            torch.ops.kb_nano_fp8_moe.router_gemm(x2, weight, out)
        else:
            _ops.moe_router_gemm(x2, weight, out)
        return out if hidden_states.dim() == 2 else out.view(*hidden_states.shape[:-1], weight.shape[0])


class MoeRouterTopk(nn.Module):
    """``forward(logits, top_k, scoring="softmax", bias=None, num_groups=1,
    topk_groups=1, renormalize=True, scale=1.0, index_dtype=torch.int32) ->
    (topk_weights, topk_ids)``: bf16, fp16 or fp32 logits ``[..., E]``, E <= 1024,
    to fp32 weights and ids ``[..., top_k]``, top_k <= 64.

    ``scoring``: "softmax" over the experts or "sigmoid" of each.  ``bias`` (fp32
    [E], finite) is added to the scores for the choice alone, never to the
    weights.  With ``num_groups`` > 1 (consecutive experts, at most 64 groups) the
    experts of the best ``topk_groups`` groups compete; a group ranks by its
    largest score, with a bias by the sum of its two largest biased scores.
    ``renormalize``: the chosen experts' weights sum to one; ``scale`` multiplies
    them.

    Experts come in descending order of their (biased) scores, equal ones with
    the lower id first.  An expert of logit -inf or NaN is taken only where no
    other is left, with weight 0; a token of such experts alone gets weights 0."""

    def forward(self, logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None,
                num_groups: int = 1, topk_groups: int = 1, renormalize: bool = True, scale: float = 1.0,
                index_dtype: torch.dtype = torch.int32) -> tuple[torch.Tensor, torch.Tensor]:
        if _ops._host is not None and not torch.compiler.is_compiling():
            out = _ops._host.router_topk(logits, top_k, scoring, bias, num_groups, topk_groups, renormalize, scale, index_dtype)
            if out is not None:
                return out
        l2 = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
        weights = torch.empty(l2.shape[0], top_k, dtype=torch.float32, device=l2.device)
        ids = torch.empty(l2.shape[0], top_k, dtype=index_dtype, device=l2.device)
        if torch.compiler.is_compiling():
            torch.ops.kb_nano_fp8_moe.router_topk(l2, top_k, scoring, bias, num_groups, topk_groups, renormalize, scale,
                                                  weights, ids)
        else:
            _ops.moe_router_topk(l2, top_k, scoring, bias, num_groups, topk_groups, renormalize, scale, weights, ids)
        if logits.dim() == 2:
            return weights, ids
        return weights.view(*logits.shape[:-1], top_k), ids.view(*logits.shape[:-1], top_k)
