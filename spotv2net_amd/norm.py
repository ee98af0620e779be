"""Layer norm over the last dimension on hand-written gfx950 kernels.

``layer_norm(x, weight, bias, eps)`` and ``LayerNorm`` take float32, bfloat16
and float16 tensors with rows of up to 16,384 elements; weight and bias are
float32 or of the input's type.  Statistics and sums are float32.  Rows may have
any stride (a column slice of a wider buffer is read in place).  The reference
normalises only its inputs (``standardize``, utils/models.py:79-83, BatchNorm);
``GATModel(layer_norm=True)`` normalises every GAT layer's output with these.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import library  # noqa: F401  (registers torch.ops.sv2n.layer_norm)


def _check_device(x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"spotv2net_amd runs layer_norm only on a ROCm GPU (got a "
                           f"{x.device.type} tensor); there is no CPU fallback")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (biased variance); differentiable once in x, weight and bias.  The result is
    dense and of x's type."""
    _check_device(x)
    return torch.ops.sv2n.layer_norm(x, weight, bias, eps)[0]


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` over one dimension (same constructor, parameters
    and state_dict) whose forward and backward run on the sv2n kernels."""

    def __init__(self, normalized_shape, *args, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises the last dimension only (got normalized_shape "
                             f"{self.normalized_shape})")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError(f"LayerNorm({self.normalized_shape[0]}): got rows of {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)
