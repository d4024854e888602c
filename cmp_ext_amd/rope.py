"""Tables for the position rotation of `qk_norm_rope`.

The rotation reads its cosines and sines from fp32 tables, so that every way of scaling positions
is a table: made once, kept by the program, shared by all layers.
"""
from __future__ import annotations

import math

import torch

__all__ = ["rope_table"]


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
               original_positions: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
               attention_factor: float | None = None, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), each float32 [max_positions, rotary_dim / 2], of position * f_i with
    f_i = base^(-2 i / rotary_dim); computed in float64.

    scaling, for contexts `factor` times those of training:
      "none"    f_i as above;
      "linear"  positions divided by factor (position interpolation);
      "ntk"     base multiplied by factor^(rotary_dim / (rotary_dim - 2)): the highest frequency
                stays, the lowest is divided by factor;
      "yarn"    frequencies that turn more than beta_fast times within original_positions stay, those
                that turn less than beta_slow times are divided by factor, those between are mixed
                linearly by their turns, and both tables are multiplied by attention_factor
                (0.1 ln(factor) + 1 unless given).  Implementations that mix linearly over the
                index i instead, between the indices of the two bounds, turn those between by other
                frequencies (up to a factor of 3 for 128, factor 16 and 4096 positions): a model
                that was trained with one needs its own tables, which `qk_norm_rope` takes as well.
    """
    if max_positions < 0:
        raise ValueError(f"rope_table: max_positions must not be negative, got {max_positions}")
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rope_table: rotary_dim must be even and not negative, got {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"rope_table: base must be positive and finite, got {base}")
    if not (factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"rope_table: factor must be at least 1 and finite, got {factor}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"rope_table: unknown scaling {scaling!r}")
    if scaling == "none" and factor != 1:
        raise ValueError("rope_table: factor needs a scaling")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-2 * i / max(rotary_dim, 1))
    size = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not original_positions or original_positions <= 0:
            raise ValueError("rope_table: yarn needs original_positions")
        if not beta_fast > beta_slow > 0:
            raise ValueError("rope_table: yarn needs beta_fast > beta_slow > 0")
        turns = original_positions * freq / (2 * math.pi)
        kept = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
        freq = freq * kept + freq / factor * (1 - kept)
        size = 0.1 * math.log(factor) + 1 if attention_factor is None else attention_factor
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
    return (angle.cos() * size).float().to(device), (angle.sin() * size).float().to(device)
