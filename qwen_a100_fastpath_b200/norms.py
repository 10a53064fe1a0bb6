"""The residual update between two blocks of a decoder layer with the norms on both sides of it, in one pass
(``qf_residual_norm`` in ``libqf_b200``), and the norms of queries and keys for each head with the position rotation
(``qf_qk_norm_rope``).

The reference plugin leaves norms to vLLM; ``w8a16.w8a16_mm_rmsnorm`` fuses the plain one into the int8 GEMM.  Here it
stands alone, with the optional norm after the block, the block's gate and the residual scale, and can hand the next
block-scaled fp8 product its quantized activations directly.  The norms inside the attention, which come with the rotation,
can hand the keys and values to the 4-bit cache in the same way.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import LIB, check, load_torch_ops, refused_out

load_torch_ops()
_norm = torch.ops.qf_b200.residual_norm.default
_norm_out = torch.ops.qf_b200.residual_norm_out.default
_rope = torch.ops.qf_b200.qk_norm_rope.default
_rope_kv4 = torch.ops.qf_b200.qk_norm_rope_kv4.default

GATE_ACTS = {"none": _lib.QF_GATE_NONE, "sigmoid": _lib.QF_GATE_SIGMOID, "silu": _lib.QF_GATE_SILU}


def residual_norm(x: torch.Tensor, residual: torch.Tensor | None, pre_weight: torch.Tensor | None, eps: float = 1e-6,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, gate_act: str = "none",
                  residual_scale: float = 1.0, weight_offset: float = 0.0, quantize: bool = False,
                  residual_out: torch.Tensor | None = None):
    """``(h, r)`` for the block output ``x`` bf16 ``[..., H]`` (H <= 16384, fewer than 2^31 rows), in fp32 inside:

    * ``u = x``, or with ``post_weight`` bf16 ``[H]`` ``u = x * rsqrt(mean(x^2) + eps) * (post_weight + weight_offset)``;
    * ``v = u``, or with ``gate`` (bf16, broadcast to x's shape) ``v = u * act(gate)``, ``gate_act`` one of "none" (the
      gate itself), "sigmoid", "silu";
    * ``r = residual + residual_scale * v`` in the residual's type (bf16 or fp32); ``residual=None`` stands for zeros and
      gives a bf16 ``r``;
    * ``h = r * rsqrt(mean(r^2) + eps) * (pre_weight + weight_offset)`` from the unrounded ``r``: bf16 ``[..., H]``, or
      with ``quantize`` the pair ``(q, scale)`` that ``fp8.fp8_quantize`` would make of the unrounded ``h``; ``None`` where
      ``pre_weight`` is ``None``.

    ``residual_out`` receives ``r``; it may be ``residual`` itself (updated in place) and must share no other memory with an
    input (refused as ``fp8.fp8_block_mm`` does).  The same rules on devices, streams and errors as in ``fp8``."""
    act = GATE_ACTS.get(gate_act)
    if act is None:
        raise ValueError(f"gate_act must be one of {tuple(GATE_ACTS)}, got {gate_act!r}")
    if residual_out is None:
        h, s, r = _norm(x, residual, pre_weight, post_weight, gate, act, residual_scale, weight_offset, eps, quantize)
    else:
        try:
            h, s = _norm_out(x, residual, pre_weight, post_weight, gate, act, residual_scale, weight_offset, eps, quantize,
                             residual_out)
        except ValueError as e:
            raise refused_out(e) from None
        r = residual_out
    return ((h, s) if quantize else h), r


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 positions: torch.Tensor | None, cos_sin: torch.Tensor | None, eps: float = 1e-6,
                 weight_offset: float = 0.0, interleaved: bool = False, v: torch.Tensor | None = None, cache=None,
                 slots: torch.Tensor | None = None):
    """``(q, k)`` bf16 ``[tokens, heads, D]`` (any strides, views of the qkv product's rows; D <= 512) normalised for each
    head and rotated, in fp32 inside and rounded once:

    * ``y = x``, or with the weight (bf16 ``[D]``) ``y = x * rsqrt(mean(x^2) + eps) * (weight + weight_offset)``;
    * the first R values of a head turn: with ``cos, sin = cos_sin[position].chunk(2)`` of ``cos_sin`` fp32 or bf16
      ``[max_positions, R]`` (``None``: no rotation) and ``a, b = y[:R / 2], y[R / 2:R]``, or ``y[0:R:2], y[1:R:2]`` where
      ``interleaved``: ``a * cos - b * sin`` and ``b * cos + a * sin``.  ``positions`` int64 ``[tokens]``; one outside the
      table makes the turned values NaN.

    With ``cache`` (a ``kv4.KV4Cache``), ``v`` and ``slots`` the keys, rounded to bf16, and ``v`` go to the cache as
    ``kv4.kv4_write`` writes them, and the result is ``(q, None)``.  The same rules on devices, streams and errors as in
    ``kv4``."""
    if (cache is None) != (v is None) or (cache is None) != (slots is None):
        raise ValueError("qk_norm_rope: cache, v and slots go together")
    if cache is None:
        return _rope(q, k, q_weight, k_weight, positions, cos_sin, weight_offset, eps, interleaved)
    try:
        return _rope_kv4(q, k, q_weight, k_weight, positions, cos_sin, weight_offset, eps, interleaved, v, slots, *cache), None
    except ValueError as e:
        raise refused_out(e) from None


def residual_norm_status(device=None) -> int:
    """Read and clear the device's sticky error flag of ``residual_norm`` (``QF_OK``, or ``QF_ERR_TIMEOUT`` after a bounded
    wait for a row inside a launch expired; the rows were then read another way and the results are valid); synchronises
    the device's current stream."""
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        st = ctypes.c_int(0)
        stream = torch.cuda.current_stream().cuda_stream
        check("qf_residual_norm_status", LIB.qf_residual_norm_status(stream, ctypes.byref(st)))
        return st.value
