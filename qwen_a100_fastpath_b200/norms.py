"""The residual update between two blocks of a decoder layer with the norms on both sides of it, in one pass
(``qf_residual_norm`` in ``libqf_b200``).

The reference plugin leaves norms to vLLM; ``w8a16.w8a16_mm_rmsnorm`` fuses the plain one into the int8 GEMM.  Here it
stands alone, with the optional norm after the block, the block's gate and the residual scale, and can hand the next
block-scaled fp8 product its quantized activations directly.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import LIB, check, load_torch_ops, refused_out

load_torch_ops()
_norm = torch.ops.qf_b200.residual_norm.default
_norm_out = torch.ops.qf_b200.residual_norm_out.default

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


def residual_norm_status(device=None) -> int:
    """Read and clear the device's sticky error flag of ``residual_norm`` (``QF_OK``, or ``QF_ERR_TIMEOUT`` after a bounded
    wait for a row inside a launch expired; the rows were then read another way and the results are valid); synchronises
    the device's current stream."""
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        st = ctypes.c_int(0)
        stream = torch.cuda.current_stream().cuda_stream
        check("qf_residual_norm_status", LIB.qf_residual_norm_status(stream, ctypes.byref(st)))
        return st.value
