"""The step between two blocks of a layer that is normed before and after its
blocks, with a gate on the block's output and a scale on the residual:

    p         = RMSNorm(input, post_weight)            (input itself without one)
    residual' = residual_scale * residual + gate * p   (in the rows' type)
    normed    = RMSNorm(residual', weight)

No counterpart in kb_nano; the modules stand beside ``RMSNormFP8Quant`` and
``FusedAddRMSNormFP8Quant``.  One launch a call: rows are read once and stay in
registers over both norms (up to 16384 columns; longer rows are read three
times).  bf16, fp16 or fp32 rows, all tensors of one type, any hidden size that
is a multiple of 8.  For inference, as the rest of the package: outputs carry
no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _ops
from .rmsnorm_quant import _outputs


def _gate_rows(gate: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor | None:
    """``gate`` (broadcast against ``like``) as [T, H] with a column stride of 0 or 1."""
    if gate is None:
        return None
    try:
        g = gate.expand(like.shape)
    except RuntimeError:
        raise ValueError(f"gated_add_rmsnorm: a gate of {tuple(gate.shape)} does not broadcast to the input's "
                         f"{tuple(like.shape)}") from None
    g = g if g.dim() == 2 else g.reshape(-1, like.shape[-1])
    return g if g.stride(1) in (0, 1) else g.contiguous()


def _run(input, residual, weight, post_weight, gate, residual_scale, eps, rows, codes):
    if _ops._host is not None and not torch.compiler.is_compiling():
        got = _ops._host.gated_norm(input, residual, weight, post_weight, gate, residual_scale, eps, rows, codes)
        if got is not None:   # the plain case in one native step
            return got
    if residual.shape != input.shape:
        raise ValueError(f"gated_add_rmsnorm: residual {tuple(residual.shape)} and input {tuple(input.shape)} differ")
    H = input.shape[-1]
    x2, r2 = (input, residual) if input.dim() == 2 else (input.reshape(-1, H), residual.reshape(-1, H))
    res = torch.empty(x2.shape, dtype=input.dtype, device=input.device)
    out = torch.empty(x2.shape, dtype=input.dtype, device=input.device) if rows else None
    q, s = _outputs(x2) if codes else (None, None)
    args = (x2, r2, weight, post_weight, _gate_rows(gate, input), residual_scale, eps, res, out, q, s)
    if torch.compiler.is_compiling():
        torch.ops.kb_nano_norm.gated_add_rmsnorm(*args)
    else:
        _ops.gated_add_rmsnorm(*args)
    if input.dim() != 2:
        res, out = res.view(input.shape), out.view(input.shape) if rows else None
    return out, q, s, res


class GatedAddRMSNorm(nn.Module):
    """``forward(input, residual, weight, post_weight=None, gate=None,
    residual_scale=1.0, eps=1e-6) -> (normed, residual')``, both new tensors of
    input's shape ``[..., H]``.  ``gate`` broadcasts against input: [H] a value for
    each channel, [..., 1] for each token, [..., H] for each element.  Others ([B, 1, H],
    one for each sequence) are spread to a [T, H] of their own first: one launch and
    two such tensors of traffic more."""

    def forward(self, input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
        normed, _, _, res = _run(input, residual, weight, post_weight, gate, residual_scale, eps, True, False)
        return normed, res


class GatedAddRMSNormFP8Quant(nn.Module):
    """``forward(input, residual, weight, post_weight=None, gate=None,
    residual_scale=1.0, eps=1e-6, with_rows=False) -> (output_fp8, output_scales,
    residual')``: as ``GatedAddRMSNorm``, the normed rows quantized as
    ``RMSNormFP8Quant`` does (output_fp8 [num_tokens, H] float8_e4m3fn,
    output_scales [num_tokens, num_groups] float32 column-major, from the unrounded
    values).  ``with_rows`` adds the normed rows themselves as a fourth output, for
    a router or adapters beside the FP8 product."""

    def forward(self, input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                eps: float = 1e-6, with_rows: bool = False) -> tuple[torch.Tensor, ...]:
        normed, q, s, res = _run(input, residual, weight, post_weight, gate, residual_scale, eps, with_rows, True)
        return (q, s, res, normed) if with_rows else (q, s, res)
