"""CPU definition of the 4-bit paged cache and of what a step does around it: the oracle of ``kv4.py``, ``paged.py`` and
``norms.qk_norm_rope``.

The quantizer is defined in fp32 operations (include/qf_b200.h), so that ``quantize`` and ``values`` are exact; everything
else is in float64 over the values that the inputs and the cache stand for.
"""
from __future__ import annotations

import numpy as np

GROUP = 64


def round_bf16(x: np.ndarray) -> np.ndarray:
    """Nearest bf16 number of float64 ``x``, ties to even, as float64 (8 significant bits, exponents down to 2^-126 and
    steps of 2^-133 below)."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(x)
    with np.errstate(invalid="ignore", over="ignore"):
        step = np.ldexp(1.0, np.maximum(e, -125) - 8)
        r = np.rint(x / step) * step
    return np.where(np.abs(r) >= 2.0 ** 128, np.copysign(np.inf, x), r)


def quantize(x: np.ndarray):
    """Nibbles uint8 ``[..., D]`` and (step, offset) float64 ``[..., D / 64, 2]`` (bf16 numbers) of bf16 values ``x``."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        s = round_bf16(((hi - lo) * (np.float32(1) / np.float32(15))).astype(np.float32)).astype(np.float32)
        c = round_bf16((lo - np.float32(16) * s).astype(np.float32)).astype(np.float32)
        bad = ~((np.abs(lo) < 2.0 ** 126) & (np.abs(hi) < 2.0 ** 126))
        q = np.rint(((g - c[..., None]).astype(np.float32) / s[..., None]).astype(np.float32))
        n = np.where(s[..., None] > 0, np.clip(q, 16, 31) - 16, 0)
    n = np.where(bad[..., None], 0, n).astype(np.uint8).reshape(x.shape)
    sc = np.stack([s, c], -1).astype(np.float64)
    sc[bad] = np.nan
    return n, sc


def pack(n: np.ndarray) -> np.ndarray:
    return (n[..., 0::2] | n[..., 1::2] << 4).astype(np.uint8)


def unpack(codes: np.ndarray) -> np.ndarray:
    return np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def values(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 ``[..., D]`` of bytes ``[..., D / 2]`` and (step, offset) ``[..., D / 64, 2]``."""
    n = unpack(codes).astype(np.float64).reshape(*scale.shape[:-1], GROUP)
    s, c = (np.asarray(scale, np.float64)[..., i, None] for i in range(2))
    return round_bf16((n + 16) * s + c).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def attention(query, cache, seq_lens, block_table, q_len, scale):
    """``(out, spread, spread_scores)`` float64: the result ``[B * q_len, H, D]``, ``sum_j w_j |v_j|`` of each element, and
    the largest ``scale * sum_d |q_d k_d|`` of each row.  ``cache``: codes k, v and scales as numpy arrays."""
    k4, v4, ks, vs = cache
    n_pages, hkv, page, _ = k4.shape
    B, H, D = len(seq_lens), query.shape[1], query.shape[2]
    g = H // hkv
    out, spread = np.zeros((B * q_len, H, D)), np.zeros((B * q_len, H, D))
    top = np.zeros((B * q_len, H))
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), block_table.shape[1] * page)
        pos = np.arange(n)
        entry = block_table[b, pos // page].astype(np.int64) if n else np.zeros(0, np.int64)
        there = (entry >= 0) & (entry < n_pages)
        pos, entry = pos[there], entry[there]
        for j in range(hkv):
            k = values(k4[entry, j, pos % page], ks[entry, j, pos % page])
            v = values(v4[entry, j, pos % page], vs[entry, j, pos % page])
            for i in range(q_len):
                seen = pos <= int(seq_lens[b]) - q_len + i
                if not seen.any():
                    continue
                qr = query[b * q_len + i, j * g:(j + 1) * g].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    x = scale * (qr @ k[seen].T)
                    w = np.exp(x - x.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    rows = (b * q_len + i, slice(j * g, (j + 1) * g))
                    out[rows], spread[rows] = w @ v[seen], w @ np.abs(v[seen])
                    top[rows] = abs(scale) * (np.abs(qr) @ np.abs(k[seen]).T).max(-1)
    return out, spread, top


def norm_rope(x, weight, positions, cos_sin, eps, offset, interleaved):
    """``(y, size)`` float64: the rotated rows ``[T, H, D]`` and ``|a cos| + |b sin|`` of each element."""
    y = np.asarray(x, np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (np.asarray(weight, np.float64) + offset)
    y = y.copy()
    size = np.abs(y)
    if cos_sin is not None:
        rot = cos_sin.shape[1]
        ok = (positions >= 0) & (positions < cos_sin.shape[0])
        row = np.where(ok[:, None], cos_sin[np.where(ok, positions, 0)] if cos_sin.shape[0] else np.nan, np.nan)
        c, s = row[:, None, :rot // 2], row[:, None, rot // 2:]
        ia = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
        ib = ia + (1 if interleaved else rot // 2)
        a, b = y[..., ia], y[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia], size[..., ib] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, size


def step_maps(query_lens, past_lens, block_table, page, num_tokens, free_pages=None, free_head=0):
    """``(query_start, seq_lens, positions, slots, free_head, block_table)`` by one loop over requests and tokens."""
    table = [list(map(int, r)) for r in block_table]
    start, seq, pos, slots = [0], [], [0] * num_tokens, [-1] * num_tokens
    head = max(int(free_head), 0)
    for r, (q, past) in enumerate(zip(query_lens, past_lens)):
        q, past, width = max(int(q), 0), max(int(past), 0), len(table[r])
        if free_pages is not None:
            for col in range(min(-(-past // page), width), min(-(-(past + q) // page), width)):
                table[r][col] = int(free_pages[head]) if head < len(free_pages) else -1
                head += 1
        for t in range(q):
            i, p = start[-1] + t, past + t
            if i >= num_tokens:
                break
            pos[i] = p
            if p // page < width and table[r][p // page] >= 0:
                slots[i] = table[r][p // page] * page + p % page
        start.append(start[-1] + q)
        seq.append(past + q)
    return start, seq, pos, slots, head, table
