"""The 8-bit paged KV cache: rows quantised as they are written, read back,
and attended (``paged_decode_attention`` and ``paged_tree_attention`` with
scales).

A row, one token of one KV head, is held as 8-bit codes and an fp32 scale:
scale = amax / 448 (float8_e4m3fn) or amax / 127 (int8), code = the nearest
number of the type (ties to even) to row / scale.  It stands for code * scale.
A row that holds a NaN or an infinity stands for NaN.

Pages of 64 tokens, with whole 16-byte units along the dimension that each
product of attention reduces over:
  k [num_pages, Hkv, D/16, 64, 16]    units of 16 features
  v [num_pages, Hkv, 4, D, 16]        units of 16 tokens
  k_scale, v_scale [num_pages, Hkv, 64] float32
The reference has no counterpart.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .attention import PAGE

_APPEND = torch.ops.spyre.kv_quant_append.default
_ROTARY_APPEND = torch.ops.spyre.rotary_kv_quant_append.default
_READ = torch.ops.spyre.kv_quant_read.default
CACHE_DTYPES = (torch.float8_e4m3fn, torch.int8)


def _tokens(t: torch.Tensor, one: bool) -> torch.Tensor:
    return t.unsqueeze(1) if one else t


def kv_append_quantized(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                        slots: torch.Tensor) -> None:
    """Quantises token t of sequence b (k_new / v_new float16 [B, T, Hkv, D],
    or [B, Hkv, D] for one token) into slot slots[b, t] (int32 [B, T] or [B]) of
    the sequence's pages, in one launch.  Negative slots are skipped; those
    past the block table, or in pages that it does not name validly, are
    dropped.  Two tokens of a call must not share a slot."""
    one = k_new.dim() == 3
    try:
        _APPEND(_tokens(k_new, one), _tokens(v_new, one), k_cache, v_cache, k_scale, v_scale, block_table,
                _tokens(slots, one))
    except RuntimeError as e:
        raise _lib.library_error(e) from None


def rotary_kv_append_quantized(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                               v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                               block_table: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                               frequencies: torch.Tensor, amplitude: float = 1.0,
                               interleaved: bool = False) -> torch.Tensor:
    """``kv_append_quantized`` with the positions (int32 or int64, [B, T] or
    [T]; [B] for one token) rotated into K first, and into q [B, T, Hq, D] (or
    [B, Hq, D]), whose rotation is returned: one launch for what a step does
    before attention.  As ``rotary_embedding``, but K's rotated values are
    quantised without a rounding to float16 between.  The rotated features are a
    multiple of 16."""
    one = q.dim() == 3
    try:
        out = _ROTARY_APPEND(_tokens(q, one), _tokens(k_new, one), _tokens(v_new, one), k_cache, v_cache, k_scale,
                             v_scale, block_table, _tokens(slots, one), _tokens(positions, one), frequencies,
                             float(amplitude), interleaved)
    except RuntimeError as e:
        raise _lib.library_error(e) from None
    return out.squeeze(1) if one else out


def kv_read_quantized(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                      block_table: torch.Tensor, lens: torch.Tensor, length: int,
                      start: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V, float16 [B, Hkv, length, D]: row i is token start[b] + i (start
    int32 [B], default 0) while that is below lens[b] (int32 [B]), else zeros.
    Tokens of pages that the block table does not name validly are NaN."""
    try:
        return _READ(k_cache, v_cache, k_scale, v_scale, block_table, lens, length, start)
    except RuntimeError as e:
        raise _lib.library_error(e) from None


class QuantizedKVCache:
    """An 8-bit paged KV cache in the layouts above."""

    def __init__(self, num_pages: int, Hkv: int, D: int, dtype: torch.dtype = torch.float8_e4m3fn, device=None):
        if D not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if dtype not in CACHE_DTYPES:
            raise ValueError(f"cache dtype must be float8_e4m3fn or int8 (got {dtype})")
        device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.num_pages, self.Hkv, self.D, self.dtype = num_pages, Hkv, D, dtype
        codes = {"dtype": torch.uint8, "device": device}
        self.k = torch.zeros((num_pages, Hkv, D // 16, PAGE, 16), **codes).view(dtype)
        self.v = torch.zeros((num_pages, Hkv, PAGE // 16, D, 16), **codes).view(dtype)
        self.k_scale = torch.ones((num_pages, Hkv, PAGE), dtype=torch.float32, device=device)
        self.v_scale = torch.ones((num_pages, Hkv, PAGE), dtype=torch.float32, device=device)

    @property
    def tensors(self) -> tuple:
        """(k, v, k_scale, v_scale), as the functions take them."""
        return self.k, self.v, self.k_scale, self.v_scale

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor,
               slots: torch.Tensor) -> None:
        kv_append_quantized(k_new, v_new, *self.tensors, block_table, slots)

    def rotary_append(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor,
                      slots: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor,
                      amplitude: float = 1.0, interleaved: bool = False) -> torch.Tensor:
        return rotary_kv_append_quantized(q, k_new, v_new, *self.tensors, block_table, slots, positions, frequencies,
                                          amplitude, interleaved)

    def read(self, block_table: torch.Tensor, lens: torch.Tensor, length: int,
             start: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        return kv_read_quantized(*self.tensors, block_table, lens, length, start)
