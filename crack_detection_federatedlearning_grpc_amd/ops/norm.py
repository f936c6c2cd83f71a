"""Layer norm (kernels: layer_norm.hip; checks and autograd: csrc/block_ops.cpp)."""
from __future__ import annotations

from typing import Optional

import torch

from .._native_loader import hip


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-3) -> torch.Tensor:
    """Keras LayerNormalization over the last axis (its epsilon default), differentiable in x, weight and bias.

    x: (..., C), float32, bfloat16 or float16, C up to 8,192; rows at one stride (a channel slice of a wider map) are
    read in place. weight, bias: fp32 (C,), as all weights of ``ops``; ones / zeros if not given. Statistics and the
    weights' gradients are fp32. Returns x's shape and type, contiguous.
    """
    return hip().layer_norm(x, weight, bias, eps)
