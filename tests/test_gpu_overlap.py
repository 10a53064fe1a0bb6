"""Outputs that share memory with inputs, through the views that the operators take: rows of larger buffers."""
from __future__ import annotations

import pytest

from tests.test_gpu_fp8 import make_weight, make_x

pytestmark = pytest.mark.gpu


def refused(f):
    """Refused as an argument (and as torch's own operators do), before anything is written."""
    for kind in (ValueError, RuntimeError):
        with pytest.raises(kind, match="single memory location"):
            f()


def test_residual_out(dev):
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    M, H = 6, 256
    pre = torch.ones(H, dtype=torch.bfloat16, device=dev)
    x0, r0 = make_x(dev, M, H, seed=1), make_x(dev, M, H, seed=2)
    h, r = residual_norm(x0, r0, pre)

    def call(x, residual, out, pre=pre, **kw):
        return residual_norm(x, residual, pre, residual_out=out, **kw)

    buf = torch.zeros(M + 1, H + 8, dtype=torch.bfloat16, device=dev)
    refused(lambda: call(x0, buf[:M, :H], buf[1:, :H]))                    # the next row's residual
    refused(lambda: call(x0, buf[1:, :H], buf[:M, :H]))
    refused(lambda: call(x0, buf[:M, :H], buf[:M, 8:]))                    # the same rows, other columns
    refused(lambda: call(buf[:M, :H], r0, buf[1:, :H]))
    refused(lambda: call(x0, r0, buf[:M, :H], gate=buf[1:, :H], gate_act="silu"))
    refused(lambda: call(x0, r0, buf[:M, :H], gate=buf[2, :H]))            # one row for all tokens
    refused(lambda: call(x0, r0, buf[:M, :H], gate=buf[:M, 100:101]))      # one value for each token
    refused(lambda: call(x0, r0, buf[:M, :H], pre=buf[3, 4:4 + H]))
    refused(lambda: call(x0[:3], buf[:3, :H], buf[1:4, :H]))
    assert not buf.any()
    # neighbours that share no element: other rows of one buffer, other columns, one between the other's
    two = torch.zeros(M, 2, H, dtype=torch.bfloat16, device=dev)
    for res, out in ((two[:, 0], two[:, 1]), (two[:, 1], two[:, 0])):
        res.copy_(r0)
        h2, r2 = call(x0, res, out)
        assert r2 is out and torch.equal(h2, h) and torch.equal(out, r) and torch.equal(res, r0)
    rows = torch.zeros(2 * M, H + 8, dtype=torch.bfloat16, device=dev)
    rows[:M, :H] = r0
    assert torch.equal(call(x0, rows[:M, :H], rows[M:, :H])[1], r)
    wide = torch.zeros(3 * M, H, dtype=torch.bfloat16, device=dev)         # every third row beside every second
    wide[1::3] = r0
    assert torch.equal(call(x0[:2], wide[1:5:3], wide[0:4:2])[1], r[:2])
    refused(lambda: call(x0[:3], wide[1:8:3], wide[0:6:2]))                # rows 1 4 7 and 0 2 4
    # in place, through another view of the same rows
    one = r0[:1].clone()
    assert torch.equal(call(x0[:1], one, one.as_strided((1, H), (7 * H, 1)))[1], r[:1])
    assert torch.equal(one, r[:1])


def test_product_out(dev):
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    M, N, K = 5, 256, 256
    a, sa = fp8_quantize(make_x(dev, M, K, seed=3))
    w, sw, _ = make_weight(dev, N, K)
    y = fp8_block_mm(a, sa, w, sw)
    mem = torch.zeros(64, 1024, dtype=torch.uint8, device=dev)             # rows of 1024 bytes

    def bf16(rows, col):
        return mem.view(torch.bfloat16)[rows, col // 2:col // 2 + N]

    av = mem.view(torch.float8_e4m3fn)[8:8 + M, 512:512 + K]
    av.copy_(a)
    sv = mem.view(torch.float32)[20:20 + M, 4:6]
    sv.copy_(sa)
    wv = mem.view(torch.float8_e4m3fn)[30:30 + 32, :K]                     # 32 weight rows
    before = mem.clone()
    assert torch.equal(fp8_block_mm(av, sv, w, sw), y)
    refused(lambda: fp8_block_mm(av, sa, w, sw, out=bf16(slice(8, 8 + M), 512)))
    refused(lambda: fp8_block_mm(av, sa, w, sw, out=bf16(slice(12, 12 + M), 256)))   # its first row on the last of a's
    refused(lambda: fp8_block_mm(a, sv, w, sw, out=bf16(slice(16, 16 + M), 0)))
    refused(lambda: fp8_block_mm(a, sa, wv.t(), sw[:1], out=mem.view(torch.bfloat16)[57:57 + M, :32]))
    bias = mem.view(torch.bfloat16)[40, :N]
    refused(lambda: fp8_block_mm(a, sa, w, sw, bias=bias, out=bf16(slice(38, 38 + M), 0)))
    refused(lambda: fp8_block_mm(a, sa, w, mem.view(torch.float32)[0:2, 0:2], out=bf16(slice(0, M), 0)))
    assert torch.equal(mem, before)
    out = bf16(slice(8, 8 + M), 0)                                         # beside a in the same rows
    assert torch.equal(fp8_block_mm(av, sa, w, sw, out=out), y)
    assert torch.equal(av.view(torch.uint8), a.view(torch.uint8))
