"""Drafted tokens checked against the target's probabilities: the step after
``paged_tree_attention`` and ``paged_latent_attention`` over them.  The reference
has no counterpart."""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_VERIFY = torch.ops.spyre.verify_drafts.default


def verify_drafts(draft_tokens: torch.Tensor, target_probs: torch.Tensor, uniforms: torch.Tensor,
                  draft_probs: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None,
                  draft_lens: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which of the drafted tokens [B, T] (int32 or int64) are kept, and the token
    behind them, so that the result is distributed as the target's own samples.

    target_probs [B, T + 1, V] (float32, float16 or bfloat16): row 0 behind the
    context, row i + 1 behind drafted token i.  uniforms float32 [B, T + 1] in [0,
    1): one for each drafted token's test, the last for the drawn token.

    A chain: token i is kept while u_i q_i(x_i) < p_i(x_i), with q = ``draft_probs``
    [B, T, V] that it was drawn from, or u_i < p_i(x_i) without; behind the first
    rejected one a token is drawn from max(p - q, 0), or from p without the
    rejected token.  A tree: ``parents`` int32 [B, T], parents[b, i] < i the drafted
    token that token i continues, -1 the context's end; the children of the last
    kept token are tried in their order, each against what the rejected ones before it
    leave of p (no draft_probs).  If no token is left to try, one is drawn from the
    last row.  ``draft_lens`` int32 [B]: drafted tokens of each sequence (default T).

    The drawn token is the lowest whose running sum exceeds u_T times the total,
    in 64-bit sums.  Returns tokens [B, T + 1] (the kept ones, the drawn one, then
    -1), the number kept (int32 [B]) and their indices (int32 [B, T], then -1).  One
    launch; at most 1024 drafted tokens."""
    try:
        return _VERIFY(draft_tokens, target_probs, uniforms, draft_probs, parents, draft_lens)
    except RuntimeError as e:
        raise _lib.library_error(e) from None
