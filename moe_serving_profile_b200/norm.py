"""The norm in front of a router and its experts.

``AddRMSNorm`` adds the attention output to the residual stream, norms the sum
and, for experts that compute in 8 bits, returns the normed rows in their
8-bit form as well: the codes of the fp32 rows, before their rounding to bf16::

    n = norm(attn_out, residual)
    _, weights, indices = router(n.out)
    y = experts(n.out, indices, weights, rows=n.rows)
"""

from __future__ import annotations

import torch
from torch import nn

from moe_serving_profile_b200 import ops


class AddRMSNorm(nn.Module):
    """``weight * h / sqrt(mean(h^2) + eps)`` of ``h = x + residual`` in fp32,
    rounded once. ``quant``: "fp8" (rows of W8A8 FP8 experts), "int8" (rows of
    int8 experts and projections) or None."""

    def __init__(self, hidden_size: int, eps: float = 1e-6, quant: str | None = None):
        super().__init__()
        if quant not in ops.QUANT:
            raise ValueError(f"quant must be one of {tuple(ops.QUANT)}, got {quant!r}")
        if hidden_size % 8:
            raise NotImplementedError(f"hidden size ({hidden_size}) must be a multiple of 8")
        self.hidden_size, self.eps, self.quant = hidden_size, eps, quant
        self.weight = nn.Parameter(torch.ones(hidden_size), requires_grad=False)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, *, inplace: bool = False,
                normed: bool = True) -> ops.NormOut:
        """``x`` and ``residual`` are bf16 [T, H]; ``inplace`` updates
        ``residual`` instead of returning a new one."""
        if inplace and residual is None:
            raise ValueError("an update in place needs a residual")
        return ops.add_rmsnorm(x, self.weight, self.eps, residual=residual,
                               residual_out=residual if inplace else None, quant=self.quant, normed=normed)
