"""A self-attention block on NHWC maps, composed of the layers of ``ops``."""
from __future__ import annotations

from typing import Optional

import torch

from .attention import attention
from .norm import layer_norm
from .rotary import grid_positions, rotary


def self_attention2d(x: torch.Tensor, norm_weight: torch.Tensor, norm_bias: torch.Tensor, w_qkv: torch.Tensor,
                     w_out: torch.Tensor, heads: int, b_qkv: Optional[torch.Tensor] = None,
                     b_out: Optional[torch.Tensor] = None, kv_heads: Optional[int] = None,
                     mask: Optional[torch.Tensor] = None, theta: float = 10000.0, eps: float = 1e-3) -> torch.Tensor:
    """x + conv1x1(attention(conv1x1(layer_norm(x)))) on an NHWC bf16 map, every pixel a token whose query and key are
    turned by its row and column (half of a head's channels each).

    w_qkv: (1, 1, C, (heads + 2 * kv_heads) * D), w_out: (1, 1, heads * D, C), fp32, Keras Conv2D layout (``conv2d``:
    channel counts in multiples of 32); D a multiple of 8 up to 128. mask: bool, True = may be attended, broadcastable
    to (B, heads, H * W, H * W), e.g. (B, 1, 1, H * W) for the valid pixels of padded images.
    """
    from . import conv2d
    if x.dim() != 4:
        raise ValueError(f"self_attention2d: x must be (B, H, W, C), got {tuple(x.shape)}")
    kv = heads if kv_heads is None else kv_heads
    B, H, W, C = x.shape
    total = heads + 2 * kv
    if heads < 1 or kv < 1 or w_qkv.dim() != 4 or tuple(w_qkv.shape[:3]) != (1, 1, C) or w_qkv.shape[3] % total:
        raise ValueError(f"self_attention2d: w_qkv {tuple(w_qkv.shape)} does not make {heads} query and 2 x {kv} key "
                         f"and value heads of {C} channels")
    D = w_qkv.shape[3] // total
    if D % 8 or tuple(w_out.shape) != (1, 1, heads * D, C):
        raise ValueError(f"self_attention2d: w_out {tuple(w_out.shape)} does not take {heads} heads of {D} channels "
                         f"to {C}")
    qkv = conv2d(layer_norm(x, norm_weight, norm_bias, eps), w_qkv, b_qkv).view(B, H * W, total, D)
    pos = grid_positions(H, W, device=x.device)
    qk = rotary(qkv[:, :, :heads + kv], pos, (D // 2, D // 2), theta)
    y = attention(qk[:, :, :heads], qk[:, :, heads:], qkv[:, :, heads + kv:], mask)
    return x + conv2d(y.reshape(B, H, W, heads * D), w_out, b_out)


__all__ = ["self_attention2d"]
