"""The maps of a step on a paged cache, built on the GPU from the requests' lengths (``qf_step_maps`` in ``libqf_b200``).

The reference plugin gets them ready-made from vLLM's model runner, which makes them on the host; ``kv4.kv4_write``,
``norms.qk_norm_rope``, ``kv4.kv4_attention`` and ``spec_attn.gqa_packed_spec_attention`` take them as they are made here,
without a copy from the host between the steps of a captured graph.  The same rules on devices, streams and errors as in
``kv4``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import load_torch_ops, refused_out

load_torch_ops()
_maps = torch.ops.qf_b200.step_maps.default
_maps_grow = torch.ops.qf_b200.step_maps_grow.default


class StepMaps(NamedTuple):
    """``query_start`` int32 ``[B + 1]``: where each request's tokens begin in the step, and their number; ``seq_lens`` int32
    ``[B]``: the lengths after the step; ``positions``, ``slots`` int64 ``[num_tokens]``; ``free_head`` int32 ``[1]``: the first
    page of the free list that is left, ``None`` where none was given.  Results of one type are pieces of one allocation
    without a common element: one that is kept (or saved) keeps the others' memory, a ``clone()`` does not."""
    query_start: torch.Tensor
    seq_lens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    free_head: torch.Tensor | None


def step_maps(query_lens: torch.Tensor, past_lens: torch.Tensor, block_table: torch.Tensor, page_size: int,
              num_tokens: int, free_pages: torch.Tensor | None = None, free_head: torch.Tensor | None = None) -> StepMaps:
    """The maps of a step of ``B`` requests (at most 16384) with ``query_lens`` int32 ``[B]`` new tokens behind
    ``past_lens`` int32 ``[B]`` cached ones (negative ones count as zero), for ``num_tokens`` tokens, the step's own or the
    larger number it is padded to.  Token ``i`` of request ``r`` has the position ``p = past_lens[r] + i`` and the slot
    ``block_table[r, p // page_size] * page_size + p % page_size`` of ``block_table`` int32 ``[B, max_pages]``, or -1 where
    the table has no page for it (an entry below zero, or a position behind its width).  Tokens behind the last request's get
    position 0 and slot -1.

    With ``free_pages`` int32 ``[F]`` and ``free_head`` int32 ``[1]`` the tables grow first, in place: entries
    ``ceil(past / page_size)`` to ``ceil((past + query) / page_size) - 1`` of each request (within ``max_pages``) receive the
    pages of ``free_pages`` from index ``free_head`` on, in the requests' order, -1 where the list has run out; the result's
    ``free_head`` counts all that was asked for, so that one above ``F`` tells how many pages are missing.  The same call
    again gives the same result: ``free_head`` itself is not changed."""
    if (free_pages is None) != (free_head is None):
        raise ValueError("step_maps: free_pages and free_head go together")
    if free_pages is None:
        return StepMaps(*_maps(query_lens, past_lens, block_table, page_size, num_tokens), None)
    try:
        return StepMaps(*_maps_grow(query_lens, past_lens, block_table, page_size, num_tokens, free_pages, free_head))
    except ValueError as e:
        raise refused_out(e) from None
