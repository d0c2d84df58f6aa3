"""The paged latent cache and its attention.

Models with latent attention project a token to one latent vector c (``rank``
features), from which every head's keys and values are expanded, and one rotated
key r (64 features) that all heads share; only (c, r) is cached.  Two forms of the
same attention:

* over the cache itself (``paged_latent_attention``), for decode steps and drafted
  tokens: with head h's weights W_k [D, rank] and W_v [D, rank], q . (W_k c) =
  (W_k^T q) . c, so q goes in as W_k^T q [.., rank], and the output sum_t p_t c_t [.., rank] is
  multiplied by W_v behind it;
* expanded (``latent_attention``), for prompts: k = W_k c and v = W_v c of every head
  are products of the program's, over rows of the prompt or of ``latent_read``.

Pages of 64 tokens, in sticks of 64 features: cache float16 [num_pages, (rank +
64) / 64, 64, 64], the layout of an fp16 K page (``k_page_layout``) of one head of
rank + 64 features.  The reference has no counterpart.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .attention import PAGE, k_page_layout

ROPE = 64
RANKS = (256, 512)
_APPEND = torch.ops.spyre.latent_append.default
_READ = torch.ops.spyre.latent_read.default
_PAGED = torch.ops.spyre.paged_latent_attention.default
_EXPANDED = torch.ops.spyre.latent_attention.default


def latent_append(latent: torch.Tensor, k_rope: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes rows of latent float16 [..., rank] and k_rope [..., 64] (rotated) into
    slots (int64 [...]: 64 page + token, as ``plan_pages`` gives them), in one launch.
    Slots outside of the cache, -1 among them, are dropped.  Two rows of a call
    must not share a slot."""
    try:
        _APPEND(latent, k_rope, cache, slots)
    except RuntimeError as e:
        raise _lib.library_error(e) from None


def latent_read(cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, length: int,
                start: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Latent vectors [B, length, rank] and rotated keys [B, length, 64]: row i is
    token start[b] + i (start int32 [B], default 0) while that is below lens[b]
    (int32 [B]), else zeros.  Tokens of pages that the block table does not name
    validly are NaN."""
    try:
        return _READ(cache, block_table, lens, length, start)
    except RuntimeError as e:
        raise _lib.library_error(e) from None


def paged_latent_attention(q: torch.Tensor, q_rope: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                           context_lens: torch.Tensor, scale: float, tree_mask: Optional[torch.Tensor] = None,
                           draft_lens: Optional[torch.Tensor] = None, max_context_len: Optional[int] = None,
                           return_lse: bool = False):
    """softmax(scale (q . c + q_rope . r)) c for every head over the tokens (c, r) of
    the paged cache.  Sequence b has context_lens[b] of them (int32 [B]) and, appended
    behind them, draft_lens[b] (int32 [B], default T) new ones; query i of q [B, T, H,
    rank] and q_rope [B, T, H, 64] (float16; [B, H, ...] for one token) attends the context
    and the new tokens j with tree_mask[b, i, j] (bool [B, T, T] or [T, T]), or j <= i
    without a mask: a decode step's query its own token as well.

    scale is that of the expanded keys, usually (D + 64)^-1/2.  Returns out [B, T, H,
    rank] and, with ``return_lse``, the fp32 logsumexp [B, T, H].  Rows i >=
    draft_lens[b], and rows that attend nothing (or only scores of -inf), are zeros with
    logsumexp -inf; what a row does not attend does not reach it; a row that attends a
    new token with a NaN or an infinity is NaN.  ``max_context_len`` bounds context_lens
    (if omitted it is read from them, which synchronises); longer contexts, and pages
    that the block table does not name validly, make the sequence NaN."""
    one = q.dim() == 3
    if one:
        q, q_rope = q.unsqueeze(1), q_rope.unsqueeze(1)
    try:
        o, lse = _PAGED(q, q_rope, cache, block_table, context_lens, float(scale), tree_mask, draft_lens,
                        -1 if max_context_len is None else int(max_context_len))
    except RuntimeError as e:
        raise _lib.library_error(e) from None
    if one:
        o, lse = o.squeeze(1), lse.squeeze(1)
    return (o, lse) if return_lse else o


def latent_attention(q: torch.Tensor, q_rope: torch.Tensor, k: torch.Tensor, k_rope: torch.Tensor, v: torch.Tensor,
                     context_lens: torch.Tensor, new_lens: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, return_lse: bool = False):
    """Causal attention of every head with its own keys k [B, keys, H, D], the
    rotated ones k_rope [B, keys, 64] that all heads share behind them, and values v [B,
    keys, H, D] (float16, any strides with features next to each other: halves of one
    projection's output go in as they are).  Sequence b has context_lens[b] keys
    (int32 [B]) before its new_lens[b] (default T) queries; query i of q [B, T, H, D] and
    q_rope [B, T, H, 64] attends the keys up to context_lens[b] + i.  scale defaults
    to (D + 64)^-1/2; D is 64 or 128.

    Returns out [B, T, H, D] and, with ``return_lse``, the fp32 logsumexp [B, T, H].  Rows
    i >= new_lens[b], and rows whose scores are all -inf, are zeros with logsumexp -inf;
    what a row does not attend does not reach it, keys behind the sequence's last among
    it, and a NaN or an infinity in a value reaches only that feature of the rows that
    attend it.  A sequence with more context and queries than there are keys is NaN."""
    try:
        o, lse = _EXPANDED(q, q_rope, k, k_rope, v, context_lens, new_lens, None if scale is None else float(scale))
    except RuntimeError as e:
        raise _lib.library_error(e) from None
    return (o, lse) if return_lse else o


class LatentKVCache:
    """A paged latent cache in the layout above."""

    def __init__(self, num_pages: int, rank: int = 512, device=None):
        if rank not in RANKS:
            raise ValueError(f"rank must be one of {RANKS} (got {rank})")
        device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.num_pages, self.rank = num_pages, rank
        self.pages = torch.zeros((num_pages, (rank + ROPE) // 64, PAGE, 64), dtype=torch.float16, device=device)
        self.layout = k_page_layout(num_pages, 1, rank + ROPE)

    def append(self, latent: torch.Tensor, k_rope: torch.Tensor, slots: torch.Tensor) -> None:
        latent_append(latent, k_rope, self.pages, slots)

    def read(self, block_table: torch.Tensor, lens: torch.Tensor, length: int,
             start: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        return latent_read(self.pages, block_table, lens, length, start)

    def attend(self, q: torch.Tensor, q_rope: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
               scale: float, tree_mask: Optional[torch.Tensor] = None, draft_lens: Optional[torch.Tensor] = None,
               max_context_len: Optional[int] = None, return_lse: bool = False):
        return paged_latent_attention(q, q_rope, self.pages, block_table, context_lens, scale, tree_mask, draft_lens,
                                      max_context_len, return_lse)
