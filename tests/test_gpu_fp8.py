"""Block-scaled fp8 layers on the GPU (fp8.py over qf_fp8_quantize / qf_fp8_block_gemm) against the float64 oracle.

Tolerances.  Quantizer without the gate: the definition's fp32 operations are single IEEE ones, so values and scales are
bit-identical.  With the gate: v carries a relative error of at most 16 * 2^-24 (exp, sum, quotient, product), so a scale
is off by at most 18 * 2^-24 and a value by half an e4m3 step (2^-4 of it, 2^-10 below 2^-6) plus that.  Product: a
product of two e4m3 values is exact; a tensor-core instruction adds 32 of them to its accumulator with an error of at
most 2^-22 of the terms' magnitudes (truncation of the aligned terms at 24 bits allowed), four per group; then one
multiply-add per group, the eight warps' or CTAs' sums and the product of the two scales, half a step (2^-24) each; the
result is rounded once: half a step of its type.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import fp8_oracle as orc

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().double().cpu().numpy()


def make_x(dev, M, K, seed=0, ld=None, off=0, special=True):
    """bf16 [M, K] with row stride ld at an element offset; a zero group, an outlier and tiny values among them."""
    import torch
    ld = K if ld is None else ld
    x = np.random.RandomState(seed).standard_normal((M, K)).astype(np.float32)
    if special and K > 128:
        x[0, :128] = 0.0
        x[M - 1, K - 1] = 300.0
        x[M // 2, 128:] *= 1e-3
    buf = torch.full((M * ld + off + 8,), 7.0, dtype=torch.bfloat16, device=dev)
    v = buf[off:off + M * ld].view(M, ld)[:, :K]
    v.copy_(torch.from_numpy(x))
    return v


def make_weight(dev, N, K, seed=1, ldw=None):
    """(w_t [K, N] view, w_scale, float64 values [N, K]): random e4m3 bytes without NaN, block scales around 2^-10."""
    import torch
    rs = np.random.RandomState(seed)
    b = rs.randint(0, 256, size=(N, K)).astype(np.uint8)
    b[(b & 127) == 127] = 0
    ldw = (K + 15) // 16 * 16 if ldw is None else ldw
    rows = np.full((N, ldw), 0x7F, np.uint8)          # NaN in the padding: it must never be used
    rows[:, :K] = b
    s = (rs.random_sample((orc.groups(N), orc.groups(K))) * 2e-3 + 1e-4).astype(np.float32)
    w = torch.from_numpy(rows).to(dev).view(torch.float8_e4m3fn)[:, :K].t()
    return w, torch.from_numpy(s).to(dev), orc.E4M3[b]


def sum_error(K):
    """Error of an output's sums relative to the magnitudes of its terms."""
    return 4 * 2.0 ** -22 + (orc.groups(K) + 8 + 3) * 2.0 ** -24


def check_mm(got, y, mag, K, bf16=True):
    err = np.abs(f64(got) - y)
    half = 2.0 ** -8 if bf16 else 2.0 ** -24
    tol = half * np.abs(y) + (1 + half) * sum_error(K) * mag + 1e-38
    assert err.shape == tol.shape
    worst = np.max(err / tol)
    assert worst <= 1.0, worst


# ---- quantizer -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,K,ld,off", [
    (1, 1, None, 0), (1, 128, None, 0), (1, 5120, None, 0), (5, 17408, None, 0), (3, 127, None, 0), (3, 129, None, 0),
    (7, 1000, 1032, 0), (7, 1000, 1001, 3), (130, 640, None, 1), (700, 1160, None, 0), (33, 8192, 8200, 8),
])
def test_quantize(dev, M, K, ld, off):
    from qwen_a100_fastpath_b200.fp8 import fp8_quantize
    x = make_x(dev, M, K, seed=M + K, ld=ld, off=off)
    q, s = fp8_quantize(x)
    assert q.shape == (M, K) and s.shape == (M, orc.groups(K)) and (M == 1 or q.stride(0) % 16 == 0)
    q_o, s_o = orc.quantize(f64(x))
    assert np.array_equal(s.cpu().numpy().view(np.uint32), s_o.view(np.uint32))
    assert np.array_equal(f64(q), q_o)


@pytest.mark.parametrize("M,K,ld,off", [(1, 64, None, 0), (5, 17408, None, 0), (3, 129, None, 0), (9, 1000, 2016, 0),
                                        (9, 1001, 2003, 1), (300, 640, None, 0)])
def test_quantize_silu_mul(dev, M, K, ld, off):
    from qwen_a100_fastpath_b200.fp8 import fp8_quantize
    x = make_x(dev, M, 2 * K, seed=M + K, ld=ld, off=off)
    x[0, 0] = -120.0                                   # exp(120) overflows fp32: the gate closes
    x[M - 1, :K].clamp_(min=-30)
    q, s = fp8_quantize(x, silu_mul=True)
    v = orc.silu_mul(f64(x))
    e_v = 16 * 2.0 ** -24
    for g in range(orc.groups(K)):
        c = slice(g * 128, min(K, g * 128 + 128))
        s_o = np.maximum(np.abs(v[:, c]).max(axis=1), 448 * 2.0 ** -60) / 448
        got_s = f64(s)[:, g]
        assert np.all(np.abs(got_s - s_o) <= (e_v + 2.0 ** -23) * s_o)
        err = np.abs(f64(q)[:, c] * got_s[:, None] - v[:, c])
        tol = np.maximum(2.0 ** -4 * np.abs(v[:, c]), 2.0 ** -10 * s_o[:, None]) * (1 + 2.0 ** -18) + \
            4 * e_v * np.abs(v[:, c]) + 1e-38
        assert np.all(err <= tol), np.max(err / tol)


def test_quantize_not_finite(dev):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_quantize
    x = make_x(dev, 4, 300, seed=3)
    x[1, 140] = float("nan")
    x[2, 299] = float("-inf")
    q, s = fp8_quantize(x)
    q_o, s_o = orc.quantize(f64(x))
    assert np.array_equal(np.isnan(f64(q)), np.isnan(q_o)) and np.array_equal(np.isnan(f64(s)), np.isnan(s_o))
    ok = ~np.isnan(q_o)
    assert np.array_equal(f64(q)[ok], q_o[ok]) and torch.isinf(s[2, 2])


def test_quantize_shapes(dev):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_quantize
    x = make_x(dev, 12, 200, seed=5)
    q, s = fp8_quantize(x)
    q3, s3 = fp8_quantize(x.view(3, 4, 200))
    assert q3.shape == (3, 4, 200) and s3.shape == (3, 4, 2)
    assert np.array_equal(f64(q3).reshape(12, 200), f64(q)) and torch.equal(s3.view(12, 2), s)
    q1, s1 = fp8_quantize(x[5])
    assert q1.shape == (200,) and s1.shape == (2,) and np.array_equal(f64(q1), f64(q)[5])
    qt, st = fp8_quantize(x.t().contiguous().t())      # column-major rows are copied
    assert np.array_equal(f64(qt), f64(q)) and torch.equal(st, s)
    qe, se = fp8_quantize(x[5].expand(6, 200))         # one row for all
    assert np.array_equal(f64(qe), np.repeat(f64(q)[5:6], 6, 0)) and qe.stride(0) != 0
    q0, s0 = fp8_quantize(x[:0])
    assert q0.shape == (0, 200) and s0.shape == (0, 2)


# ---- product -------------------------------------------------------------------------------------------------
SHAPES = [
    (1, 16, 128), (1, 1, 1), (1, 5120, 8192), (2, 129, 17), (3, 17, 1000), (5, 1536, 2048), (8, 300, 640), (9, 200, 1160),
    (16, 1024, 5120), (17, 1000, 200), (31, 64, 384), (33, 640, 520), (64, 2048, 1024), (72, 1280, 5120), (127, 257, 129),
    (128, 256, 256), (129, 384, 1000), (200, 4352, 4096), (333, 2600, 1160), (512, 512, 2176), (700, 130, 77), (1000, 1, 300),
    (256, 2304, 128), (1030, 3000, 1024),
    (40, 96, 1), (100, 1, 16), (16, 9500, 130), (7, 9480, 300), (6, 5000, 1023), (90, 512, 20000), (4500, 136, 256),
]


@pytest.mark.parametrize("bias,out", [(False, "bf16"), (True, "f32")])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_block_mm(dev, M, N, K, bias, out):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    a, sa = fp8_quantize(make_x(dev, M, K, seed=M + N))
    w, sw, wv = make_weight(dev, N, K, seed=N + K)
    b = torch.randn(N, device=dev).to(torch.bfloat16) if bias else None
    y = fp8_block_mm(a, sa, w, sw, bias=b, out_dtype=torch.float32 if out == "f32" else torch.bfloat16)
    assert y.shape == (M, N) and y.dtype == (torch.float32 if out == "f32" else torch.bfloat16)
    ref, mag = orc.block_mm(f64(a), f64(sa), wv, f64(sw), f64(b) if bias else None)
    check_mm(y, ref, mag, K, out == "bf16")


@pytest.mark.parametrize("M", [3, 40, 300])
def test_block_mm_strides(dev, M):
    """Strided and misaligned activation rows, scales in any order or shared, padded weight rows, a strided result whose
    other columns and rows stay as they were."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    N, K = 200, 520
    a, sa = fp8_quantize(make_x(dev, M, K, seed=M))
    w, sw, wv = make_weight(dev, N, K, ldw=1024)
    ref, mag = orc.block_mm(f64(a), f64(sa), wv, f64(sw))
    base = fp8_block_mm(a, sa, w, sw, out_dtype=torch.float32)
    check_mm(base, ref, mag, K, False)
    wide = torch.full((M, 1024), 0x7F, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    wide[:, 32:32 + K] = a
    odd = torch.full((M * 521 + 1,), 0x7F, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)[1:].view(M, 521)[:, :K]
    odd.copy_(a)
    for a2, sa2, sw2 in ((wide[:, 32:32 + K], sa.t().contiguous().t(), sw.t().contiguous().t()), (odd, sa, sw)):
        assert torch.equal(fp8_block_mm(a2, sa2, w, sw2, out_dtype=torch.float32), base)
    one = torch.full((1, 1), 0.5, device=dev).expand(M, orc.groups(K))
    y = fp8_block_mm(a, one, w, sw, out_dtype=torch.float32)
    ref1, mag1 = orc.block_mm(f64(a), np.full((M, orc.groups(K)), 0.5), wv, f64(sw))
    check_mm(y, ref1, mag1, K, False)
    for dt in (torch.bfloat16, torch.float32):
        buf = torch.full((M + 2, N + 13), 3.0, dtype=dt, device=dev)
        out = buf[1:M + 1, 5:5 + N]
        assert fp8_block_mm(a, sa, w, sw, out=out) is out
        check_mm(out, ref, mag, K, dt == torch.bfloat16)
        out.fill_(3.0)
        assert (buf == 3.0).all()


@pytest.mark.parametrize("M", [2, 50, 400])
def test_block_mm_not_finite(dev, M):
    """A NaN or an infinite scale stays in its own token's row."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    x = make_x(dev, M, 300, seed=2)
    good, gs = fp8_quantize(x)
    w, sw, _ = make_weight(dev, 144, 300)
    base = fp8_block_mm(good, gs, w, sw)
    x[1, 7] = float("nan")
    y = fp8_block_mm(*fp8_quantize(x), w, sw)
    assert torch.isnan(y[1]).all()
    keep = [i for i in range(M) if i != 1]
    assert torch.equal(y[keep], base[keep])
    x[1, 7] = float("inf")
    y = fp8_block_mm(*fp8_quantize(x), w, sw)
    assert not torch.isfinite(y[1]).any() and torch.equal(y[keep], base[keep])


@pytest.mark.parametrize("M", [1, 12, 90])
def test_block_mm_exact_small_integers(dev, M):
    """Small integers and power-of-two scales: every sum is exact in fp32, so the result is bit-exact."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm
    N, K = 272, 700
    rs = np.random.RandomState(4)
    ai, wi = rs.randint(-8, 9, (M, K)), rs.randint(-8, 9, (N, K))
    sa = 2.0 ** rs.randint(-2, 3, (M, orc.groups(K)))
    sw = 2.0 ** rs.randint(-2, 3, (orc.groups(N), orc.groups(K)))

    def rows(v):
        r = torch.zeros((v.shape[0], 704), dtype=torch.float8_e4m3fn, device=dev)
        r[:, :K] = torch.from_numpy(v).float().to(dev).to(torch.float8_e4m3fn)
        return r[:, :K]

    y = fp8_block_mm(rows(ai), torch.from_numpy(sa).float().to(dev), rows(wi).t(), torch.from_numpy(sw).float().to(dev),
                     out_dtype=torch.float32)
    assert np.array_equal(f64(y), orc.block_mm(ai, sa, wi, sw)[0])


@pytest.mark.parametrize("M", [4, 70])
def test_block_mm_far_offsets(dev, M):
    """Row strides whose offsets pass 2^31 bytes in the activations, the weight and the result."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    N, K = 33, 256
    a, sa = fp8_quantize(make_x(dev, M, K, seed=9))
    w, sw, wv = make_weight(dev, N, K)
    step = (2 ** 31 // min(M, N) + 4096) // 16 * 16
    far_a = torch.empty(((M - 1) * step + K,), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    far_a = far_a.as_strided((M, K), (step, 1))
    far_a.copy_(a)
    far_w = torch.empty(((N - 1) * step + K,), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    far_w = far_w.as_strided((N, K), (step, 1))
    far_w.copy_(w.t())
    far_y = torch.empty(((M - 1) * step + N,), dtype=torch.bfloat16, device=dev).as_strided((M, N), (step, 1))
    fp8_block_mm(far_a, sa, far_w.t(), sw, out=far_y)
    assert torch.equal(far_y, fp8_block_mm(a, sa, w, sw))


def test_block_mm_repeats(dev):
    """The same call twice gives the same bits (nothing is summed in an order that varies)."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_linear
    for M, N, K in ((1, 5120, 8192), (16, 1024, 5120), (72, 1280, 5120), (300, 2600, 1160)):
        x = make_x(dev, M, K, seed=M)
        w, sw, _ = make_weight(dev, N, K)
        y = fp8_block_linear(x, w, sw)
        for _ in range(3):
            assert torch.equal(fp8_block_linear(x, w, sw), y)


# ---- linear layer --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,N,K,ld,off,bias", [
    (1, 5120, 17408, None, 0, False), (1, 96, 1, None, 0, True), (4, 1000, 130, 136, 0, True), (5, 640, 1001, 1003, 1, False),
    (8, 512, 5120, None, 0, False), (13, 2048, 1160, None, 0, True), (16, 10240, 640, 648, 8, True), (17, 384, 5120, None, 0, False),
    (48, 1280, 2048, None, 0, True), (300, 640, 1160, None, 0, False),
])
def test_block_linear(dev, M, N, K, ld, off, bias):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_linear
    x = make_x(dev, M, K, seed=M + K, ld=ld, off=off)
    w, sw, wv = make_weight(dev, N, K)
    b = torch.randn(N, device=dev).to(torch.bfloat16) if bias else None
    y = fp8_block_linear(x, w, sw, b)
    q, s = orc.quantize(f64(x))                        # bit-identical to the layer's own quantization
    ref, mag = orc.block_mm(q, s, wv, f64(sw), f64(b) if bias else None)
    check_mm(y, ref, mag, K)


def test_first_call_in_a_capture():
    """A process whose first calls are captured ones (nothing that a call sets up once needs an eager call before)."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from qwen_a100_fastpath_b200.fp8 import fp8_block_linear, fp8_status
from qwen_a100_fastpath_b200.norms import residual_norm
dev = torch.device('cuda', 0)
g = torch.Generator(device=dev).manual_seed(1)
w = torch.randn(512, 640, device=dev, generator=g).to(torch.float8_e4m3fn).t()
sw = torch.rand(4, 5, device=dev, generator=g)
n = torch.ones(640, device=dev, dtype=torch.bfloat16)
xs = [torch.randn(m, 640, device=dev, generator=g).to(torch.bfloat16) for m in (3, 12, 50, 4000)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = [fp8_block_linear(residual_norm(x, x, n)[0], w, sw) for x in xs]
graph.replay()
torch.cuda.synchronize()
for x, y in zip(xs, out):
    assert torch.equal(fp8_block_linear(residual_norm(x, x, n)[0], w, sw), y)
assert fp8_status() == 0
print('captured first')
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_block_linear_shapes_and_not_finite(dev):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_linear
    w, sw, _ = make_weight(dev, 256, 384)
    x = make_x(dev, 12, 384, seed=8)
    y = fp8_block_linear(x, w, sw)
    assert torch.equal(fp8_block_linear(x.view(2, 6, 384), w, sw), y.view(2, 6, 256))
    assert fp8_block_linear(x[:0], w, sw).shape == (0, 256)
    assert fp8_block_linear(x[3], w, sw).shape == (256,)
    x[4, 200] = float("nan")
    x[6, 0] = float("inf")
    z = fp8_block_linear(x, w, sw)
    keep = [i for i in range(12) if i not in (4, 6)]
    assert torch.isnan(z[4]).all() and not torch.isfinite(z[6]).any() and torch.equal(z[keep], y[keep])


# ---- refusals that need a device ------------------------------------------------------------------------------
def test_refusals(dev):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_linear, fp8_block_mm, fp8_quantize
    x = make_x(dev, 4, 256)
    a, sa = fp8_quantize(x)
    w, sw, _ = make_weight(dev, 256, 256)
    b = torch.zeros(256, dtype=torch.bfloat16, device=dev)
    cases = [
        lambda: fp8_quantize(x.half()),
        lambda: fp8_quantize(x[:, :255], silu_mul=True),
        lambda: fp8_quantize(x[:, :0]),
        lambda: fp8_quantize(x.clone().requires_grad_()),
        lambda: fp8_block_mm(a.view(torch.uint8), sa, w, sw),
        lambda: fp8_block_mm(a, sa[:, :1], w, sw),
        lambda: fp8_block_mm(a, sa.double(), w, sw),
        lambda: fp8_block_mm(a, sa.cpu(), w, sw),
        lambda: fp8_block_mm(a, sa, w[:255], sw),
        lambda: fp8_block_mm(a, sa, w.contiguous(), sw),            # not the view of weight rows
        lambda: fp8_block_mm(a, sa, w, sw[:1]),
        lambda: fp8_block_mm(a, sa, w, sw, bias=b[:100]),
        lambda: fp8_block_mm(a, sa, w, sw, bias=b.float()),
        lambda: fp8_block_mm(a[0], sa[0], w, sw),
        lambda: fp8_block_mm(a, sa, w, sw, out=torch.empty(4, 255, device=dev)),
        lambda: fp8_block_mm(a, sa, w, sw, out=torch.empty(4, 256, device=dev, dtype=torch.float16)),
        lambda: fp8_block_mm(a, sa, w, sw, out=torch.empty(256, 4, device=dev).t()),
        lambda: fp8_block_mm(a, sa, w, sw, out=torch.empty(1, 256, device=dev).expand(4, 256)),
        lambda: fp8_block_linear(x[:, :128], w, sw),
        lambda: fp8_block_linear(x.float(), w, sw),
    ]
    for i, f in enumerate(cases):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was taken")
    big = torch.empty(1 << 16, device=dev)
    sa2 = big[:8].view(4, 2)
    with pytest.raises(RuntimeError, match="single memory location"):
        fp8_block_mm(a, sa2, w, sw, out=big[:1024].view(4, 256))
    torch.cuda.synchronize(dev)


def test_no_wait_expired(dev):
    """None of the launches above (the same process) left a timeout behind."""
    from qwen_a100_fastpath_b200.fp8 import fp8_status
    assert fp8_status(dev) == 0
