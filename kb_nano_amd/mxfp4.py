"""MXFP4: quantization to 4-bit codes with a scale per 32 values, and the
linear over such weights.

Format: along K, each group of 32 values shares one power-of-two scale (E8M0,
one byte: ``torch.float8_e8m0fnu``) and each value is an e2m1 code (0, 0.5, 1,
1.5, 2, 3, 4, 6 and their negatives), two codes a byte with even k in the low
nibble.  Per group, with a the largest magnitude rounded to one mantissa bit
(ties up), the scale is 2^(floor(log2 a) - 2), at least 2^-126, and codes are
to nearest, ties to even, at most 6 in magnitude; a group that holds an
infinity or a NaN becomes NaN as a whole (scale byte 255).  The rounding in the
scale is a choice: the OCP microscaling document's own conversion leaves it out
and clips what passes 6 scales, so groups whose maximum has a mantissa of 1.75
and more get other codes there; codes and scales of either are read alike.

No counterpart in kb_nano; the modules stand beside ``PerTokenGroupQuantFp8``
and ``Fp8Linear`` and take what those take.  For inference, as the rest of the
package: outputs carry no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _ops
from ._ops import MX_GROUP


class Mxfp4Quant(nn.Module):
    """``forward(x) -> (codes, scales)``: bf16, fp16 or fp32 ``x [..., K]`` (an
    activation, or a weight at load time; K % 32 == 0) to codes uint8
    ``[..., K/2]`` and scales float8_e8m0fnu ``[..., K/32]``."""

    def forward(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        if _ops._host is not None and not torch.compiler.is_compiling():
            out = _ops._host.mx_quant(x)   # the plain case in one native step
            if out is not None:
                return out
        K = x.shape[-1]
        codes = torch.empty(*x.shape[:-1], K // 2, dtype=torch.uint8, device=x.device)
        scales = torch.empty(*x.shape[:-1], K // MX_GROUP, dtype=torch.float8_e8m0fnu, device=x.device)
        x2, c2, s2 = (x, codes, scales) if x.dim() == 2 else (_rows(x), _rows(codes), _rows(scales))
        if torch.compiler.is_compiling():
            torch.ops.kb_nano_mxfp4.quant(x2, c2, s2)
        else:
            _ops.mxfp4_quant(x2, c2, s2)
        return codes, scales


def _rows(t: torch.Tensor) -> torch.Tensor:
    n = 1
    for d in t.shape[:-1]:
        n *= d
    return t.reshape(n, t.shape[-1])


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``codes [..., K/2]`` with ``scales [..., K/32]`` as ``dtype``
    (bf16, fp16 or fp32) ``[..., K]``: a weight checked or used without the MXFP4
    product."""
    if _ops._host is not None and not torch.compiler.is_compiling():
        out = _ops._host.mx_dequant(codes, scales, _ops._QUANT_IN.get(dtype, -1))
        if out is not None:
            return out
    if scales.shape[:-1] != codes.shape[:-1]:
        raise ValueError(f"dequantize_mxfp4: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} have other rows")
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=dtype, device=codes.device)
    c2, s2, o2 = (codes, scales, out) if codes.dim() == 2 else (_rows(codes), _rows(scales), _rows(out))
    if torch.compiler.is_compiling():
        torch.ops.kb_nano_mxfp4.dequant(c2, s2, o2)
    else:
        _ops.mxfp4_dequant(c2, s2, o2)
    return out


class Mxfp4Linear(nn.Module):
    """Linear over an MXFP4 weight: ``forward(x, weight, weight_scale, bias=None)``
    quantizes bf16, fp16 or fp32 ``x [..., K]`` (K % 128 == 0) to MXFP4 and
    multiplies by ``weight`` (codes [N, K/2]) with ``weight_scale`` ([N, K/32]);
    fp32 sums, bf16 output [..., N], as ``Fp8Linear``."""

    BLOCK_SIZE = MX_GROUP

    def forward(self, x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: torch.Tensor | None = None) -> torch.Tensor:
        if _ops._host is not None and not torch.compiler.is_compiling():
            output = _ops._host.mx_linear(x, weight, weight_scale)
            if output is not None:
                return output if bias is None else output + bias
        N = weight.shape[0]
        flat = x.dim() == 2
        x2 = x if flat else _rows(x)
        output = torch.empty(x2.shape[0], N, dtype=torch.bfloat16, device=x.device)
        if torch.compiler.is_compiling():
            torch.ops.kb_nano_mxfp4.linear(x2, weight, weight_scale, output)
        else:
            _ops.mxfp4_linear(x2, weight, weight_scale, output)
        if bias is not None:
            output = output + bias
        return output if flat else output.view(*x.shape[:-1], N)
