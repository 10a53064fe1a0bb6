"""Block-scaled fp8 layers and the residual norm on the CPU: the oracle against torch's e4m3 conversions, the C ABI's
refusals before any CUDA call, and the operators' refusals of CPU tensors and of arguments that name no device."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8_oracle as orc
from qwen_a100_fastpath_b200 import _lib

FAKE = 1 << 20
LIB = _lib.LIB


# ---- the oracle ----------------------------------------------------------------------------------------------
def test_e4m3_table_is_torchs():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(t), np.isnan(orc.E4M3))
    assert np.array_equal(t[~np.isnan(t)], orc.E4M3[~np.isnan(t)])


def test_rounding_is_nearest_even():
    vals = np.sort(orc.E4M3[np.isfinite(orc.E4M3) & (orc.E4M3 >= 0)])
    vals = np.unique(vals)
    mid = (vals[1:] + vals[:-1]) / 2
    r = orc.round_e4m3(np.concatenate([vals, mid, np.nextafter(mid, 1e9), np.nextafter(mid, -1e9), -mid]))
    n = len(vals)
    assert np.array_equal(r[:n], vals)
    even = np.where(np.arange(n - 1) % 2 == 0, vals[:-1], vals[1:])   # byte order is value order: even byte wins
    assert np.array_equal(r[n:2 * n - 1], even)
    assert np.array_equal(r[2 * n - 1:3 * n - 2], vals[1:])
    assert np.array_equal(r[3 * n - 2:4 * n - 3], vals[:-1])
    assert np.array_equal(r[4 * n - 3:], -even)
    assert orc.round_e4m3(1e9) == 448.0 and np.isnan(orc.round_e4m3(np.nan))


def test_rounding_matches_torch_in_range():
    x = np.random.RandomState(0).standard_normal(20000).astype(np.float32) * np.float32(40)
    t = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(orc.round_e4m3(x.astype(np.float64)), t)


def test_oracle_quantizer_edges():
    v = np.zeros((3, 300), np.float32)
    v[1, 130] = np.nan
    v[2, 5] = np.inf
    q, s = orc.quantize(v)
    assert s.shape == (3, 3) and (s[0] == np.float32(2.0 ** -60)).all() and not q[0].any()
    assert np.isnan(s[1, 1]) and np.isnan(q[1, 128:256]).all() and not np.isnan(q[1, :128]).any()
    assert np.isinf(s[2, 0])


# ---- the C ABI ----------------------------------------------------------------------------------------------
def quantize(**kw):
    a = dict(x=FAKE, ldx=5120, M=4, K=5120, silu=0, q=FAKE, ldq=5120, scale=FAKE, lds=40, flags=0, stream=None)
    a.update(kw)
    return LIB.qf_fp8_quantize(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -2), (dict(K=-1), -2), (dict(K=_lib.QF_FP8_MAX_K + 1), -2),
    (dict(x=None), -1), (dict(q=None), -1), (dict(scale=None), -1),
    (dict(ldx=5119), -3), (dict(ldq=5119), -3), (dict(lds=39), -3),
    (dict(silu=1, ldx=10239), -3),               # gate and up: 2 K per row
    (dict(x=FAKE + 1), -4), (dict(scale=FAKE + 2), -4),
    (dict(M=1 << 30, K=512, ldx=512, ldq=512, lds=4), -2),   # more groups than a 31-bit index
])
def test_quantize_argument_validation(kw, code):
    assert quantize(**kw) == code
    assert len(LIB.qf_last_error_detail()) > 0


def gemm(**kw):
    a = dict(a=FAKE, lda=5120, sa=FAKE, sa_m=40, sa_g=1, w=FAKE, ldw=5120, sw=FAKE, sw_n=40, sw_g=1, bias=None, y=FAKE,
             ldy=1024, y_dtype=0, M=4, N=1024, K=5120, flags=0, stream=None)
    a.update(kw)
    return LIB.qf_fp8_block_gemm(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -2), (dict(N=-1), -2), (dict(K=-1), -2), (dict(K=0), -2),
    (dict(K=_lib.QF_FP8_MAX_K + 16, lda=1 << 21, ldw=1 << 21), -2),
    (dict(N=_lib.QF_MAX_N + 1, ldy=1 << 21), -2),
    (dict(a=None), -1), (dict(sa=None), -1), (dict(w=None), -1), (dict(sw=None), -1), (dict(y=None), -1),
    (dict(lda=5104), -3), (dict(ldw=5104), -3), (dict(ldy=1023), -3), (dict(sa_m=-1), -3), (dict(sw_g=-1), -3),
    (dict(a=FAKE + 8), -4), (dict(w=FAKE + 8), -4), (dict(lda=5128), -4), (dict(ldw=5128), -4),
    (dict(y=FAKE + 1), -4), (dict(y=FAKE + 2, y_dtype=1), -4), (dict(sa=FAKE + 2), -4), (dict(bias=FAKE + 1), -4),
    (dict(y_dtype=2), -8),
])
def test_gemm_argument_validation(kw, code):
    assert gemm(**kw) == code
    assert len(LIB.qf_last_error_detail()) > 0


def norm(**kw):
    a = dict(x=FAKE, ldx=512, r=FAKE, ldr=512, r_dtype=0, gate=None, gate_sm=0, gate_sh=0, act=0, post=None, pre=FAKE,
             offset=0.0, alpha=1.0, eps=1e-6, ro=FAKE, ldro=512, out=FAKE, ldo=512, scale=None, lds=0, M=4, H=512, flags=0,
             stream=None)
    a.update(kw)
    return LIB.qf_residual_norm(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), -2), (dict(H=-1), -2), (dict(H=16385, ldx=20000, ldr=20000, ldro=20000, ldo=20000), -2),
    (dict(r_dtype=2), -8), (dict(act=3), -1), (dict(act=-1), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
    (dict(eps=float("inf")), -1),
    (dict(x=None), -1), (dict(pre=None), -1), (dict(out=None), -1), (dict(out=None, pre=None, ro=None), -1),
    (dict(gate=FAKE, gate_sm=512, gate_sh=2), -3), (dict(gate=FAKE, gate_sm=-1, gate_sh=1), -3),
    (dict(ldx=511), -3), (dict(ldr=511), -3), (dict(ldro=511), -3), (dict(ldo=511), -3), (dict(scale=FAKE, lds=3), -3),
    (dict(x=FAKE + 1), -4), (dict(r=FAKE + 2, r_dtype=1), -4), (dict(pre=FAKE + 1), -4), (dict(scale=FAKE + 2, lds=4), -4),
])
def test_norm_argument_validation(kw, code):
    assert norm(**kw) == code
    assert len(LIB.qf_last_error_detail()) > 0


def test_status_needs_a_place():
    assert LIB.qf_fp8_status(None, None) == -1


def test_empty_calls_make_no_cuda_call():
    assert quantize(M=0) == 0 and quantize(K=0, ldx=0) == 0
    assert gemm(M=0) == 0 and gemm(N=0) == 0
    assert norm(M=0) == 0 and norm(H=0) == 0


# ---- the operators -----------------------------------------------------------------------------------------
def test_operators_refuse_cpu_tensors_and_bad_names():
    from qwen_a100_fastpath_b200 import fp8, norms
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    q = torch.zeros(2, 256, dtype=torch.float8_e4m3fn)
    w = torch.zeros(256, 256, dtype=torch.float8_e4m3fn).t()
    s = torch.ones(2, 2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        fp8.fp8_quantize(x)
    with pytest.raises(ValueError, match="at least one dimension"):
        fp8.fp8_quantize(torch.zeros((), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="1 to 1048576 values per row, got 0"):   # a message that formats numbers
        fp8.fp8_quantize(x[:, :0])
    with pytest.raises(ValueError, match="CUDA tensor"):
        fp8.fp8_block_mm(q, s, w, s)
    with pytest.raises(ValueError, match="CUDA tensor"):
        fp8.fp8_block_mm(q, s, w, s, out=torch.zeros(2, 256))
    with pytest.raises(ValueError, match="out_dtype"):
        fp8.fp8_block_mm(q, s, w, s, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        fp8.fp8_block_linear(x, w, s)
    with pytest.raises(ValueError, match="CUDA tensor"):
        norms.residual_norm(x, x, x[0])
    with pytest.raises(ValueError, match="gate_act"):
        norms.residual_norm(x, x, x[0], gate=x, gate_act="relu")


def test_meta_shapes():
    """Under tracing the operators answer with the shapes, types and row strides of the real call."""
    from qwen_a100_fastpath_b200 import fp8, norms
    x = torch.empty(3, 4, 1000, dtype=torch.bfloat16, device="meta")
    q, s = fp8.fp8_quantize(x)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and q.stride(-2) == 1008 and s.shape == (3, 4, 8)
    q, s = fp8.fp8_quantize(x, silu_mul=True)
    assert q.shape == (3, 4, 500) and s.shape == (3, 4, 4)
    w = torch.empty(640, 1008, dtype=torch.float8_e4m3fn, device="meta")[:, :1000].t()
    sw = torch.empty(5, 8, device="meta")
    y = fp8.fp8_block_linear(x, w, sw)
    assert y.shape == (3, 4, 640) and y.dtype == torch.bfloat16
    a, sa = fp8.fp8_quantize(x.view(12, 1000))
    assert fp8.fp8_block_mm(a, sa, w, sw, out_dtype=torch.float32).dtype == torch.float32
    r = torch.empty(3, 4, 1000, device="meta")
    (q, s), ro = norms.residual_norm(x, r, x[0, 0], quantize=True)
    assert q.shape == x.shape and s.shape == (3, 4, 8) and ro.dtype == torch.float32
    h, ro = norms.residual_norm(x, None, x[0, 0], residual_out=torch.empty_like(x))
    assert h.shape == x.shape and h.dtype == torch.bfloat16
    assert norms.residual_norm(x, r, None)[0] is None


def test_norm_status_needs_a_place():
    assert LIB.qf_residual_norm_status(None, None) == -1


@pytest.mark.parametrize("kw", [
    dict(M=_lib.QF_FP8_MAX_M + 1, K=16, lda=16, N=16, ldw=16, ldy=16),     # the last tile's rows pass 2^31
    dict(M=2 ** 31 - 1, K=16, lda=16, N=16, ldw=16, ldy=16),
    dict(M=_lib.QF_FP8_MAX_M, K=16, lda=16, N=_lib.QF_MAX_N, ldw=16, ldy=_lib.QF_MAX_N),   # more tiles than 2^31
])
def test_gemm_refuses_more_tiles_than_it_can_number(kw):
    assert gemm(**kw) == -2 and b"too large" in LIB.qf_last_error_detail()


def test_operands_are_read_by_ordinary_loads():
    """The kernels start under the tail of the kernel before them, which may still write their operands: loads that the
    hardware and the compiler may take for invariant (ld.global.nc, __ldg) are not for them."""
    from pathlib import Path
    csrc = Path(_lib.__file__).resolve().parent / "csrc"
    for name in ("qf_fp8.cuh", "qf_fp8_gemm.cu", "qf_fp8_quant.cu", "qf_norm.cu"):
        text = (csrc / name).read_text()
        assert "__ldg" not in text and "global.nc" not in text and "__restrict__" not in text, name
