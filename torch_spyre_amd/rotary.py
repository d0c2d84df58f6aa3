"""Rotary positions of q and k.

The reference rotates in its model code, by tables of cosines and sines that
its compiler lowers like any other pointwise work; this module has one kernel
for it, which forms the angles itself (no table, exact at far positions) and
is differentiable in q and k.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

_ROTARY = torch.ops.spyre.rotary.default
SCALINGS = (None, "linear", "ntk", "yarn", "llama3")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_positions: int = 8192, fast_turns: Optional[float] = None,
                       slow_turns: float = 1.0, amplitude: Optional[float] = None,
                       device=None) -> tuple[torch.Tensor, float]:
    """(frequencies, amplitude) of ``rotary_embedding``: radians per position
    of each of the rotary_dim / 2 pairs, float64 on ``device`` (default: the
    current GPU), and the factor on the rotated values.

    Plain: f_i = base^(-2i / rotary_dim).  Scaled by ``factor`` for contexts
    beyond the ``original_positions`` that the model was trained on:

    * "linear"  f_i / factor (positions interpolated);
    * "ntk"     base * factor^(rotary_dim / (rotary_dim - 2)): the slowest
                pair by factor, the fastest not at all;
    * "yarn"    pairs that make more than ``fast_turns`` (default 32) turns in
                original_positions keep f_i, those below ``slow_turns`` take
                f_i / factor, with a ramp over the pairs between; amplitude
                0.1 ln(factor) + 1 unless given;
    * "llama3"  the same with the ramp over the turns, ``fast_turns`` 4.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even (got {rotary_dim})")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS} (got {scaling!r})")
    if base <= 0 or factor <= 0 or original_positions <= 0:
        raise ValueError("base, factor and original_positions must be positive")
    fast = fast_turns if fast_turns is not None else 32.0 if scaling == "yarn" else 4.0
    if scaling in ("yarn", "llama3") and not fast > slow_turns > 0:
        raise ValueError(f"fast_turns {fast} must exceed slow_turns {slow_turns} > 0")
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** -(torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        # the (fractional) pair that makes so many turns in original_positions
        pair = [rotary_dim * math.log(original_positions / (t * 2 * math.pi)) / (2 * math.log(base))
                for t in (fast, slow_turns)]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        if amplitude is None:
            amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling == "llama3":
        turns = original_positions * f / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast - slow_turns)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    return f.to(device), 1.0 if amplitude is None else float(amplitude)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
                     amplitude: float = 1.0, interleaved: bool = False, inverse: bool = False):
    """q [B, Hq, S, D] and k [B, Hkv, S, D] (or None) with their positions
    rotated in: pair i of a head, turned by positions[b, s] * frequencies[i]
    and scaled by ``amplitude``.  Pairs are the features (i, i + R/2) of the
    first R = 2 len(frequencies), or (2i, 2i + 1) with ``interleaved``;
    features from R on are copied.  ``inverse`` turns back.

    float16, bfloat16 or float32, any strides ([B, S, H, D] tensors go in as
    their transposes); positions int32 or int64 [B, S] or [S]; frequencies
    float64, as ``rotary_frequencies`` gives them.  Returns (q, k) with the
    operands' strides where these are dense, or q alone without k.
    Differentiable in q and k, in reverse (any number of times) and forward
    mode."""
    try:
        yq, yk = _ROTARY(q, k, positions, frequencies, float(amplitude), interleaved, inverse)
    except RuntimeError as e:
        raise _lib.library_error(e) from None
    return yq if k is None else (yq, yk)
