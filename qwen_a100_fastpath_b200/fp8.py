"""Block-scaled fp8 linear layers on the B200: e4m3 weights with one fp32 scale for each block of 128 x 128, activations
quantized at run time in groups of 128 along k.

The reference plugin serves the int8 form of these layers (plugin/qwen_fastpath/w8a16.py, patches.py:84-106); checkpoints
of the same models also come with block-scaled fp8 weights, and this module is what ``w8a16.py`` is for the int8 ones.
The weight is read in place: ``w_t`` is the checkpoint's e4m3 ``[N, K]`` row-major viewed as ``[K, N]`` with stride
``(1, ldw)``, ``w_scale`` its fp32 ``[ceil(N / 128), ceil(K / 128)]`` block scales.

* ``fp8_quantize``: bf16 rows -> e4m3 rows and group scales, alone or behind the MLP's SiLU gate;
* ``fp8_block_mm``: the product of quantized activations (from here or from ``norms.residual_norm``) with a weight;
* ``fp8_block_linear``: the layer on bf16 activations.

All tensors must be CUDA tensors on one device; the work goes to that device's current stream and nothing is
synchronised, so calls can be captured into CUDA graphs.  A call that cannot be taken raises ``ValueError`` before
anything is launched; there is no CPU path, no derivative (tensors that require a gradient are refused outside
``torch.no_grad()``) and no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import LIB, check, load_torch_ops, refused_out

load_torch_ops()
_quantize = torch.ops.qf_b200.fp8_quantize.default
_mm = torch.ops.qf_b200.fp8_block_mm.default
_mm_out = torch.ops.qf_b200.fp8_block_mm_out.default
_linear = torch.ops.qf_b200.fp8_block_linear.default

FP8_BLOCK = 128


def fp8_quantize(x: torch.Tensor, silu_mul: bool = False):
    """``(q, scale)`` of bf16 ``x [..., K]``: for each row and each group of 128 consecutive k (the last may be shorter)
    ``a = max(max|v|, 448 * 2^-60)``, ``scale = a / 448`` (fp32 ``[..., ceil(K / 128)]``), ``q = e4m3(v * (448 / a))``
    rounded to nearest even (``float8_e4m3fn [..., K]``, rows 16 bytes aligned).  ``v`` is ``x``, or with ``silu_mul``
    ``silu(x[..., :K]) * x[..., K:]`` in fp32 for ``x [..., 2 K]`` (the merged gate_up output).  A NaN makes its group's
    scale and values NaN.  K <= 2^20, fewer than 2^31 groups in all."""
    return _quantize(x, silu_mul)


def fp8_block_mm(a: torch.Tensor, a_scale: torch.Tensor, w_t: torch.Tensor, w_scale: torch.Tensor,
                 bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[m, n] = sum_g a_scale[m, g] * w_scale[n // 128, g] * sum_{k in g} a[m, k] * w[n, k] (+ bias[n])``: exact e4m3
    products, fp32 sums, one rounding to ``out_dtype`` (bf16 or fp32).  ``a`` e4m3 ``[M, K]`` with fp32 ``a_scale
    [M, ceil(K / 128)]`` (any strides) as ``fp8_quantize`` returns them; ``w_t`` e4m3 ``[K, N]`` with stride ``(1, ldw)``,
    16-byte aligned, ``ldw % 16 == 0``; ``bias`` bf16 ``[N]``, added in fp32; K and N up to 2^20, M up to 2^31 - 128.  Rows
    of ``a`` that are not 16-byte aligned are copied first.  ``out`` may supply the result (it decides the type then); it
    must not share memory with an input (refused as ``_lib.QFOverlapError``, a ``ValueError``; bytes between the elements of
    an input that is not rows of adjacent elements count as its own)."""
    if out is not None:
        try:
            _mm_out(a, a_scale, w_t, w_scale, bias, out)
        except ValueError as e:
            raise refused_out(e) from None
        return out
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise ValueError("out_dtype must be torch.bfloat16 or torch.float32")
    return _mm(a, a_scale, w_t, w_scale, bias, out_dtype is torch.float32)


def fp8_block_linear(x: torch.Tensor, w_t: torch.Tensor, w_scale: torch.Tensor,
                     bias: torch.Tensor | None = None) -> torch.Tensor:
    """The linear layer of a block-scaled fp8 checkpoint on bf16 ``x [..., K]``: ``fp8_block_mm(*fp8_quantize(x), w_t,
    w_scale, bias)`` with the leading dimensions kept, bf16 ``[..., N]``."""
    return _linear(x, w_t, w_scale, bias)


def fp8_status(device=None) -> int:
    """Read and clear the device's sticky error flag of the block-scaled product (``QF_OK`` or ``QF_ERR_TIMEOUT``, after a
    bounded wait inside a launch expired); synchronises the device's current stream."""
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        st = ctypes.c_int(0)
        check("qf_fp8_status", LIB.qf_fp8_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(st)))
        return st.value
