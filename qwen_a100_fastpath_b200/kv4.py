"""The paged key / value cache held in 4 bits, and the attention that reads it, on the B200.

The reference plugin's attention reads a bf16 cache (plugin/qwen_fastpath/spec_attn.py:139-173; ``spec_attn.py`` here).
This module holds the same context in 4.5 bits a value: groups of 64 dimensions of a head of a token, a nibble for each
value and a bf16 step and offset for each group (``include/qf_b200.h`` has the exact definition).

* ``kv4_cache``: a new cache;
* ``kv4_write``: keys and values of a step into its slots (``norms.qk_norm_rope`` does it in the pass that makes the keys;
  ``paged.step_maps`` makes the slots);
* ``kv4_read``: what slots hold, as bf16;
* ``kv4_attention``: attention of a decode or verification batch over the cache.

All tensors must be CUDA tensors on one device; the work goes to that device's current stream and nothing is
synchronised, so calls can be captured into CUDA graphs.  A call that cannot be taken raises ``ValueError`` before
anything is launched; there is no CPU path, no derivative (tensors that require a gradient are refused outside
``torch.no_grad()``) and no fallback.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import load_torch_ops, refused_out

load_torch_ops()
_write = torch.ops.qf_b200.kv4_write.default
_read = torch.ops.qf_b200.kv4_read.default
_attention = torch.ops.qf_b200.kv4_attention.default
_attention_out = torch.ops.qf_b200.kv4_attention_out.default

KV4_GROUP = 64


class KV4Cache(NamedTuple):
    """``k``, ``v``: uint8 ``[pages, heads, slots, D / 2]``, the even dimension in a byte's low half; ``k_scale``,
    ``v_scale``: bf16 ``[pages, heads, slots, D / 64, 2]``, the step and the offset of each group.  D is 64, 128 or 256, a
    page may have any number of slots.  Views are fine where k and v (and their scales) have the same strides, the last
    dimensions are adjacent, and addresses and the other strides are multiples of 16 bytes (of ``D / 64`` pairs for the
    scales): of one buffer that holds keys and values (and their scales) side by side for each page, head or slot, for
    instance."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv4_cache(num_pages: int, page_size: int, num_kv_heads: int, head_size: int, device=None) -> KV4Cache:
    """A cache of zeros on ``device`` (the current CUDA device if it is not given)."""
    if head_size not in (64, 128, 256):
        raise ValueError(f"kv4_cache: head_size must be 64, 128 or 256, got {head_size}")
    if num_pages < 0 or page_size < 1 or num_kv_heads < 1:
        raise ValueError(f"kv4_cache: {num_pages} pages of {page_size} slots of {num_kv_heads} heads")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    lead = (num_pages, num_kv_heads, page_size)
    codes = [torch.zeros(*lead, head_size // 2, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.zeros(*lead, head_size // KV4_GROUP, 2, dtype=torch.bfloat16, device=device) for _ in range(2)]
    return KV4Cache(*codes, *scales)


def kv4_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: KV4Cache) -> None:
    """Quantizes ``k`` and ``v`` bf16 ``[tokens, heads, D]`` (any strides) into the slots ``slots`` int64 ``[tokens]``, slot
    ``page * page_size + offset``.  Tokens whose slot is negative (padding) or behind the cache are left out; the slots of a
    call must differ (one that is given twice holds parts of either token afterwards).  For each group of 64 values with
    ``lo`` and ``hi`` the least and the greatest: ``s = bf16((hi - lo) * (1 / 15))``, ``c = bf16(lo - 16 s)``,
    ``n = clamp(rint((x - c) / s), 16, 31) - 16`` (0 where ``s`` is 0), fp32 operations; ``n`` stands for ``bf16((n + 16) s + c)``, which is
    within ``s / 2 + s / 8 + |lo| / 256`` of ``x`` before its own rounding to bf16.  A group with a NaN, an infinity or a magnitude of
    2^126 or more becomes NaN."""
    try:
        _write(k, v, slots, *cache)
    except ValueError as e:
        raise refused_out(e) from None


def kv4_read(cache: KV4Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)`` bf16 ``[tokens, heads, D]`` that the slots ``slots`` int64 ``[tokens]`` hold; zeros for a slot that is
    negative or behind the cache."""
    return _read(*cache, slots)


def kv4_attention(query: torch.Tensor, cache: KV4Cache, seq_lens: torch.Tensor, block_table: torch.Tensor, q_len: int,
                  scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """``spec_attn.gqa_packed_spec_attention`` over a 4-bit cache: ``B = len(seq_lens)`` requests x ``q_len`` query tokens
    each (token ``b * q_len + qi``), query ``qi`` of request ``b`` attends the keys ``[0, seq_lens[b] - q_len + qi]``, this
    step's keys and values already in the cache; ``H / heads`` query heads for each key head; a row with no key gives zeros.

    ``query`` bf16 ``[>= B * q_len, H, D]`` (any strides), ``seq_lens`` int32 ``[B]``, ``block_table`` int32
    ``[>= B, max_pages]``; ``q_len * H / heads <= 64``.  Keys behind the table's width, and those on a page whose entry is
    no page of the cache (-1, for instance), do not take part.  What lies in slots that a row does not attend does not touch
    it, NaN included.  Scores, references, sums and outputs are held in fp32; the weights (relative to a reference 16 to 32
    powers of two above the row's largest score so far) are rounded to bf16 for the product with the values, while their sum
    takes them unrounded.  The sums hold up to 2^17 keys of the largest values that the cache keeps.

    Returns bf16 ``[B * q_len, H, D]``, or ``out`` (the query's shape) with its first ``B * q_len`` tokens written and the
    others left as they were; ``out`` must share no memory with an input."""
    if out is None:
        return _attention(query, *cache, seq_lens, block_table, q_len, scale)
    try:
        _attention_out(query, *cache, seq_lens, block_table, q_len, scale, out)
    except ValueError as e:
        raise refused_out(e) from None
    return out
