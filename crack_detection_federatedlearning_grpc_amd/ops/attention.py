"""Attention over token tensors (kernels: attention.hip, attention_bwd.hip; checks and autograd: csrc/block_ops.cpp).

A feature map (B, H, W, C) is read as tokens: ``x.view(B, H * W, heads, C // heads)``. Activations are bfloat16 or
float16; sums and softmax statistics are fp32. Argument errors raise ``ValueError`` / ``TypeError``.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .._native_loader import hip

Out = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor] = None,
              lengths: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
              return_lse: bool = False) -> Out:
    """softmax(scale * q k^T) v for every image and head, differentiable in q, k and v.

    q: (B, Sq, Hq, D), k, v: (B, Sk, Hkv, D); D a multiple of 8 up to 128, Hq a multiple of Hkv (query head h reads
    key head h * Hkv // Hq). Slices of a wider tensor are read in place if their rows are 16-byte aligned, else copied.
    scale: 1 / sqrt(D) if not given; positive.

    A query may attend the keys that all of these allow:
      lengths: int32 (B,): the first lengths[b] keys of image b (values are clamped to 0 .. Sk). Keys behind them are
               not read, their gradients are 0.
      mask:    bool, True = may attend, broadcastable to (B, Hq, Sq, Sk). It is packed to bits once per call; tiles in
               which it allows nothing are skipped.
      causal:  key j for query i where j <= i + Sk - Sq (the last query attends the last key).
    A query that may attend nothing gets 0, and no gradient comes from it; one whose every score is -inf gets NaN.
    Whatever a key or value holds where it is not allowed, infinities and NaN too, has no effect; an infinite value
    that may be attended shows as an infinity or NaN.

    Returns (B, Sq, Hq, D); with return_lse also the fp32 (B, Hq, Sq) log of the softmax' sum (-inf where a query may
    attend nothing; it has no gradient). The backward pass computes the probabilities again; its results do not depend
    on the order in which blocks run. It cannot be differentiated itself.
    """
    return hip().attention(q, k, v, mask, lengths, causal, scale, return_lse)


def attention_qkv(qkv: torch.Tensor, heads: int, kv_heads: Optional[int] = None, mask: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
                  return_lse: bool = False) -> Out:
    """``attention`` on one tensor (B, S, heads + 2 * kv_heads, D) of query, key and value heads, as a 1x1 convolution
    of a map makes it. Nothing is copied apart, and the gradient comes as one tensor of the same shape."""
    return hip().attention_qkv(qkv, heads, kv_heads, mask, lengths, causal, scale, return_lse)
