"""Block tables and slot maps built on the GPU from the sequences' lengths.

A paged cache's pages are handed out from a ring of free ones,
``free_pages[c % len(free_pages)]`` for taken <= c < returned, whose two counters
live in ``cursor`` (int64 [2]) and only grow; sequence b holds the first held[b]
pages of its row of the block table.  Nothing is read back: a serving loop keeps
all of it on the device and can capture its step into a graph.  The reference
has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

_PLAN = torch.ops.spyre.plan_pages.default
_RELEASE = torch.ops.spyre.release_pages.default


class PagePlan(NamedTuple):
    """What ``plan_pages`` returns: of each new token its position in the
    sequence (int32) and its slot, 64 page + token (int64; -1 where it has
    none); the pages that each sequence holds now, the ring's new cursor and, of
    packed tokens, where each sequence's begin (int32 [B + 1]; else empty)."""

    positions: torch.Tensor
    slots: torch.Tensor
    held: torch.Tensor
    cursor: torch.Tensor
    starts: torch.Tensor


def plan_pages(block_table: torch.Tensor, held: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
               free_pages: torch.Tensor, cursor: torch.Tensor, length: Optional[int] = None,
               tokens: Optional[int] = None) -> PagePlan:
    """Pages for new_lens[b] tokens behind context_lens[b] (int32 [B]) of every
    sequence: those that its held[b] (int32 [B]) lack are taken from the ring,
    sequence after sequence, and written behind the held ones in block_table
    (int32 [B, W]), in one launch.

    With ``length`` positions and slots are [B, length] (-1 from new_lens[b] on):
    ``rotary_embedding`` takes the positions, ``latent_append`` the slots, and the
    appends that take a sequence's own slots, ``kv_append_quantized`` and (a column at
    a time) ``kv_append``, torch.where(slots < 0, -1, positions).  With ``tokens`` they
    are [tokens], the sequences' tokens one after the other (-1 behind the
    last).  Where the ring or the table's row has no page left, slots are -1 and
    held[b] falls short; nothing else fails, but the table's entries from held[b] on are
    stale: no position there may be written or attended.  held and cursor are left as they
    are: keep the plan's for the next call (a captured loop copies them back).
    At most 4096 sequences."""
    if (length is None) == (tokens is None):
        raise ValueError("either length or tokens must be given")
    if (length if length is not None else tokens) < 0:
        raise ValueError("length and tokens must not be negative")
    try:
        return PagePlan(*_PLAN(block_table, held, context_lens, new_lens, free_pages, cursor,
                               -1 if length is None else int(length), -1 if tokens is None else int(tokens)))
    except RuntimeError as e:
        raise _lib.library_error(e) from None


def release_pages(block_table: torch.Tensor, held: torch.Tensor, lens: torch.Tensor, free_pages: torch.Tensor,
                  cursor: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The pages behind the first lens[b] tokens (int32 [B]; 0 for a sequence
    that has ended) go back to the ring.  Returns (held, cursor); the table
    keeps its entries, stale from held[b] on."""
    try:
        return _RELEASE(block_table, held, lens, free_pages, cursor)
    except RuntimeError as e:
        raise _lib.library_error(e) from None


class PagePool:
    """The block table of ``sequences`` rows and the ring of ``num_pages`` free
    pages, all on the device.  plan() and release() update it in place, so that
    a captured step can be replayed."""

    def __init__(self, num_pages: int, sequences: int, pages_per_seq: int, device=None):
        device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.num_pages = num_pages
        self.block_table = torch.full((sequences, pages_per_seq), -1, dtype=torch.int32, device=device)
        self.held = torch.zeros((sequences,), dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.cursor = torch.tensor([0, num_pages], dtype=torch.int64, device=device)

    def plan(self, context_lens: torch.Tensor, new_lens: torch.Tensor, length: Optional[int] = None,
             tokens: Optional[int] = None) -> PagePlan:
        p = plan_pages(self.block_table, self.held, context_lens, new_lens, self.free_pages, self.cursor, length, tokens)
        self.held.copy_(p.held)
        self.cursor.copy_(p.cursor)
        return p

    def release(self, lens: torch.Tensor) -> None:
        held, cursor = release_pages(self.block_table, self.held, lens, self.free_pages, self.cursor)
        self.held.copy_(held)
        self.cursor.copy_(cursor)
