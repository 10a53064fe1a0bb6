"""Block-scaled fp8 layers and the residual update with its norms, restated in numpy (float64 unless a step is defined in
fp32).  The reference plugin has no fp8 path; the arithmetic is the one documented in include/qf_b200.h."""
from __future__ import annotations

import numpy as np

BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = np.float32(E4M3_MAX * 2.0 ** -60)


def e4m3_table() -> np.ndarray:
    """Value of every e4m3 byte: sign, four exponent bits (bias 7), three mantissa bits; 0x7F and 0xFF are NaN."""
    b = np.arange(256)
    e, f = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b & 128, -v, v)


E4M3 = e4m3_table()


def round_e4m3(v) -> np.ndarray:
    """Nearest e4m3 value (ties to even, saturated to +-448, NaN kept) of float64 numbers."""
    v = np.asarray(v, np.float64)
    a = np.minimum(np.abs(v), E4M3_MAX)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0)
        # log2 may round up to the next binade's exponent just below a power of two
        e = np.where((2.0 ** e > a) & (e > -6), e - 1, e)
        step = 2.0 ** (e - 3)
        r = np.minimum(np.rint(a / step) * step, E4M3_MAX)
    return np.where(np.isnan(v), np.nan, np.copysign(r, v))


def groups(K: int) -> int:
    return -(-K // BLOCK)


def quantize(v: np.ndarray):
    """(q values float64, scale fp32) of fp32 rows ``v [M, K]``; every operation is the fp32 one the definition names."""
    v = np.asarray(v, np.float32)
    M, K = v.shape
    q = np.empty((M, K))
    s = np.empty((M, groups(K)), np.float32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        for g in range(groups(K)):
            c = slice(g * BLOCK, min(K, (g + 1) * BLOCK))
            a = np.maximum(np.max(np.abs(v[:, c]), axis=1), AMAX_FLOOR)      # np.maximum keeps NaN
            s[:, g] = a / np.float32(E4M3_MAX)
            q[:, c] = round_e4m3((v[:, c] * (np.float32(E4M3_MAX) / a)[:, None]).astype(np.float64))
    return q, s


def silu_mul(x: np.ndarray) -> np.ndarray:
    """float64 silu(gate) * up of merged rows [M, 2K]."""
    x = np.asarray(x, np.float64)
    K = x.shape[1] // 2
    return x[:, :K] / (1.0 + np.exp(-x[:, :K])) * x[:, K:]


def expand(scale: np.ndarray, K: int) -> np.ndarray:
    return np.repeat(np.asarray(scale, np.float64), BLOCK, axis=1)[:, :K]


def block_mm(a, a_scale, w, w_scale, bias=None):
    """(y, bound): the float64 product of values ``a [M, K]``, ``w [N, K]`` with their scales, and the sum of the
    magnitudes of its terms (what a rounding error of the sums is relative to)."""
    K, N = a.shape[1], w.shape[0]
    af = np.asarray(a, np.float64) * expand(a_scale, K)
    wf = np.asarray(w, np.float64) * np.repeat(expand(w_scale, K), BLOCK, axis=0)[:N]
    y = af @ wf.T
    mag = np.abs(af) @ np.abs(wf).T
    if bias is not None:
        y = y + np.asarray(bias, np.float64)[None, :]
        mag = mag + np.abs(np.asarray(bias, np.float64))[None, :]
    return y, mag


def act(g, kind: str):
    g = np.asarray(g, np.float64)
    if kind == "none":
        return g
    s = 1.0 / (1.0 + np.exp(-g))
    return s if kind == "sigmoid" else g * s


def rms(x, weight, offset, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + eps) * (np.asarray(weight, np.float64) + offset)[None, :]


def residual_norm(x, residual, pre, eps, post=None, gate=None, gate_act="none", alpha=1.0, offset=0.0):
    """(h, r, v) in float64 for rows [M, H]; ``h`` None without ``pre``, ``v`` the scaled block output added to r."""
    v = np.asarray(x, np.float64)
    if post is not None:
        v = rms(v, post, offset, eps)
    if gate is not None:
        v = v * act(gate, gate_act)
    v = alpha * v
    r = v if residual is None else np.asarray(residual, np.float64) + v
    return (None if pre is None else rms(r, pre, offset, eps)), r, v
