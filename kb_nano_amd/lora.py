"""Low-rank adapters of many requests beside a shared projection.

``LoraAdd`` adds each token's adapter to a projection's output; ``LoraFp8Linear``
is ``Fp8Linear`` with adapters.  Adapters are stacked: ``lora_a [L, R, K]``,
``lora_b [L, N, R]``, R a multiple of 8 up to 256 (those of smaller rank padded
with zeros), and each token names its own (``adapter_ids``); tokens of one adapter
need not be neighbours.  No counterpart in kb_nano.  For inference, as the rest
of the package: outputs carry no gradient.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _ops
from .fp8_linear import Fp8Linear


def _flat_ids(ids: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """``ids [T]`` in the order of x's rows.  Where both have several dimensions they have to be the same
    (ones aside): ids [S, B] beside x [B, S, K] would give tokens each other's adapters."""
    if ids.dim() == 1:
        return ids
    if ids.shape != x.shape[:-1]:
        mine, rows = [n for n in ids.shape if n != 1], [n for n in x.shape[:-1] if n != 1]
        if len(mine) > 1 and len(rows) > 1 and mine != rows:
            raise ValueError(f"lora_add: adapter_ids {tuple(ids.shape)} and x {tuple(x.shape)} have other rows")
    return ids.reshape(-1)


class LoraAdd(nn.Module):
    """``forward(x, base, lora_a, lora_b, adapter_ids, scaling=None, inplace=False)``:
    ``base[t] + scaling[a] * lora_b[a] @ (lora_a[a] @ x[t])`` for ``a =
    adapter_ids[t]``, ``base[t]`` for ids outside [0, L) (requests without an
    adapter, padding).  ``x [..., K]`` and ``base [..., N]`` bf16 or fp16, adapters
    of the same type, ids int32 or int64 ``[...]`` or flat ``[T]``, scaling fp32
    [L].  fp32 sums; the scaled ``lora_a[a] @ x[t]`` enters the second product as two
    bf16 numbers (2^-17 of it at most is lost), and the result is rounded once.  An
    infinity in x or an adapter leaves infinities or NaN in its tokens' rows.  Returns
    a new tensor, or with ``inplace`` base itself (which may be x, and must not overlap
    lora_b, ids or scaling)."""

    def forward(self, x: torch.Tensor, base: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, scaling: torch.Tensor | None = None, inplace: bool = False) -> torch.Tensor:
        if _ops._host is not None and not inplace and not torch.compiler.is_compiling():
            out = _ops._host.lora_add(x, base, lora_a, lora_b, adapter_ids, scaling)   # the plain case in one native step
            if out is not None:
                return out
        if x.shape[:-1] != base.shape[:-1]:
            raise ValueError(f"lora_add: x {tuple(x.shape)} and base {tuple(base.shape)} have other rows")
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        tracing = torch.compiler.is_compiling()
        if base.dim() == 2:
            b2 = base
        else:   # in place a copy of the rows would be written instead of base
            b2 = base.view(-1, base.shape[-1]) if inplace else base.reshape(-1, base.shape[-1])
        # (the compiler's ops write to no tensor that they also read)
        out = b2 if inplace and not tracing else torch.empty(b2.shape, dtype=base.dtype, device=base.device)
        args = (x2, b2, lora_a, lora_b, _flat_ids(adapter_ids, x), scaling, out)
        if tracing:
            torch.ops.kb_nano_lora.add(*args)
            if inplace:
                b2.copy_(out)
        else:
            _ops.lora_add(*args)
        return base if inplace else out if base.dim() == 2 else out.view(base.shape)


class LoraFp8Linear(nn.Module):
    """``Fp8Linear`` with adapters: ``forward(input_bf16, weight_fp8,
    weight_scale_inv, lora_a, lora_b, adapter_ids, scaling=None, bias=None)``.  The
    adapters read the bf16 input, not its FP8 codes, and are added to the
    projection's bf16 output in place; with ``linear``'s buffers installed the
    result is a view into them, as ``Fp8Linear`` returns it."""

    def __init__(self):
        super().__init__()
        self.linear = Fp8Linear()
        self.lora = LoraAdd()

    def forward(self, input_bf16: torch.Tensor, weight_fp8: torch.Tensor, weight_scale_inv: torch.Tensor,
                lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_ids: torch.Tensor,
                scaling: torch.Tensor | None = None, bias: torch.Tensor | None = None) -> torch.Tensor:
        base = self.linear(input_bf16, weight_fp8, weight_scale_inv, bias)
        return self.lora(input_bf16, base, lora_a, lora_b, adapter_ids, scaling, inplace=True)
