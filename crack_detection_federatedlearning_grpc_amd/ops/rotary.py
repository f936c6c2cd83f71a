"""Rotary positions with one to four axes (kernel: rotary.hip; checks and autograd: csrc/block_ops.cpp)."""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .._native_loader import hip


def rotary(x: torch.Tensor, positions: torch.Tensor, dims: Sequence[int], theta: float = 10000.0, joint: bool = False,
           interleaved: bool = False) -> torch.Tensor:
    """Turns the channel pairs of every head by angles of the tokens' positions; differentiable in x.

    x: (B, S, H, D), float32, bfloat16 or float16; query and key heads in one tensor take one call. positions: (A, S)
    or (A, B, S), int32, int64 or float32, one row an axis (``grid_positions``). dims: A even channel counts; the first
    sum(dims) channels of a head are rotated, the pairs of axis a following those of axis a - 1; the rest is copied.

    Pair i (counted within its axis) turns by position * theta ** (-2 i / dims[a]); with joint, i counts over all pairs
    and the exponent is -2 i / sum(dims). Pairs are (i, i + sum(dims) / 2), or (2 i, 2 i + 1) if interleaved. Angles
    are formed in 64 bits, so positions far from 0 keep their fractions of a turn.
    """
    return hip().rotary(x, positions, list(dims), theta, joint, interleaved)


def grid_positions(*sizes: int, device: Optional[torch.device] = None) -> torch.Tensor:
    """int32 (len(sizes), product) positions of the cells of a grid in row-major order: (H, W) for a map's tokens,
    (T, H, W) for a video's."""
    if not sizes or any(int(n) != n or n < 1 for n in sizes):
        raise ValueError(f"grid_positions: sizes must be positive integers, got {sizes}")
    axes = torch.meshgrid(*(torch.arange(int(n), dtype=torch.int32, device=device) for n in sizes), indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes])
