"""Rotary position tables, with one axis or several.

``build_rotary`` makes the cosines and sines that ``paged_append`` turns keys
and queries by: angle(position, pair p) = position * base^(-p / pairs),
computed in FP64 and rounded once to FP32. With ``sections`` each pair turns
by one of several positions (time, height, width of a video token):
``sections=(16, 24, 24)`` gives the first 16 pairs to axis 0, the next 24 to
axis 1 and the last 24 to axis 2, and positions are then [3, T].
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class Rotary:
    """Cosines and sines [positions, pairs] FP32, the pairs' layout and their axes."""
    cos: torch.Tensor
    sin: torch.Tensor
    interleaved: bool = False          # pairs (2p, 2p + 1) instead of (p, p + pairs)
    axis: torch.Tensor | None = None   # uint8 [pairs]: row of the positions that turns each pair


def build_rotary(max_position, dim, *, base=10000.0, interleaved=False, sections=None, device="cuda") -> Rotary:
    """Table for positions 0 .. max_position - 1 and the first ``dim`` dims of a head."""
    if max_position <= 0 or dim <= 0 or dim % 2:
        raise ValueError("max_position must be positive and dim a positive even number")
    pairs = dim // 2
    rate = float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * rate
    axis = None
    if sections is not None:
        if sum(sections) != pairs or min(sections) < 0:
            raise ValueError(f"sections {tuple(sections)} must add up to the {pairs} pairs")
        axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(torch.uint8).to(device)
    return Rotary(angle.cos().float().to(device), angle.sin().float().to(device), interleaved, axis)
