"""Block-scaled fp8 layers (fp8.py) at the largest and smallest of their sizes and arguments."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def test_more_rows_than_2_to_the_20(dev):
    """Small integers and scales of one: every sum is exact, so the products are the integer ones."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_linear, fp8_block_mm
    M, N, K = 2 ** 20 + 5, 24, 200
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randint(-8, 9, (M, K), device=dev, generator=gen).to(torch.bfloat16)
    x[:, 0], x[:, 128] = 448.0, 448.0                  # each group's largest: the quantizer's scales are one
    w = torch.zeros(N, 208, device=dev, dtype=torch.float8_e4m3fn)
    w[:, :K] = torch.randint(-8, 9, (N, K), device=dev, generator=gen).float().to(torch.float8_e4m3fn)
    w = w[:, :K]
    ones = torch.ones(1, 2, device=dev)
    want = x.float() @ w.float().t()
    a = torch.zeros(M, 208, device=dev, dtype=torch.float8_e4m3fn)[:, :K]
    a.copy_(x)
    assert torch.equal(fp8_block_mm(a, ones.expand(M, 2), w.t(), ones, out_dtype=torch.float32), want)
    assert torch.equal(fp8_block_linear(x, w.t(), ones), want.to(torch.bfloat16))


def test_too_many_rows_are_refused_first(dev):
    """Calls that are too large raise ValueError before anything is allocated, copied or launched (the inputs are one row
    that is repeated, of which a copy would not fit the device)."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_linear, fp8_block_mm, fp8_quantize
    from qwen_a100_fastpath_b200.norms import residual_norm
    x = torch.zeros(1, 256, device=dev, dtype=torch.bfloat16)
    q = torch.zeros(1, 256, device=dev, dtype=torch.float8_e4m3fn)
    w = torch.zeros(16, 256, device=dev, dtype=torch.float8_e4m3fn).t()
    s, sw = torch.ones(1, 2, device=dev), torch.ones(1, 2, device=dev)
    before = torch.cuda.memory_allocated(dev)
    for f in (lambda: fp8_quantize(x.expand(2 ** 30, 256)),                # 2^31 groups
              lambda: fp8_quantize(x.view(1, 1, 256).expand(2 ** 16, 2 ** 15, 256), silu_mul=True),
              lambda: fp8_block_linear(x.expand(2 ** 30, 256), w, sw),
              lambda: fp8_block_mm(q.expand(2 ** 31 - 127, 256), s.expand(2 ** 31 - 127, 2), w, sw),
              lambda: residual_norm(x[:, :1].expand(2 ** 31, 1), None, None)):
        with pytest.raises(ValueError, match="too many|more than"):
            f()
    # an output that does not fit is refused before unaligned rows are copied
    rows = torch.zeros(2 ** 20 * 257 + 1, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
    rows = rows[1:].view(2 ** 20, 257)[:, :256]
    base = torch.cuda.memory_allocated(dev)
    torch.cuda.reset_peak_memory_stats(dev)
    with pytest.raises(ValueError, match="out must be"):
        fp8_block_mm(rows, s.expand(2 ** 20, 2), w, sw, out=x)
    assert torch.cuda.max_memory_allocated(dev) == base
    del rows
    assert torch.cuda.memory_allocated(dev) == before


@pytest.mark.parametrize("M", [3, 16, 200])
def test_operands_written_by_the_kernel_before(dev, M):
    """Chains in which each launch, begun under the tail of the one before, reads what that one wrote over older values:
    activations, scales, bias, residual and gate.  The bits of the same calls with the device idle in between."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    from qwen_a100_fastpath_b200.norms import residual_norm
    N, K = 512, 640
    gen = torch.Generator(device=dev).manual_seed(M)

    def e4m3(*shape):
        return torch.randn(*shape, device=dev, generator=gen).to(torch.float8_e4m3fn)

    w, w2 = e4m3(N, K).t(), e4m3(K, N).t()
    sw, sw2 = torch.rand(4, 5, device=dev, generator=gen) * 0.01, torch.rand(5, 4, device=dev, generator=gen) * 0.01
    x0 = torch.randn(M, K, device=dev, generator=gen).to(torch.bfloat16)

    def chain(pause):
        def done():
            if pause:
                torch.cuda.synchronize(dev)

        r, y, z = x0.clone(), torch.zeros(M, N, device=dev), torch.zeros(M, K, device=dev, dtype=torch.bfloat16)
        kept = []
        done()
        for _ in range(12):
            h, _ = residual_norm(z, r, x0[0], gate=r, gate_act="sigmoid", residual_out=torch.empty_like(r))
            done()
            residual_norm(h, r, None, gate=h, gate_act="sigmoid", residual_out=r)   # the residual over itself
            done()
            a, s = fp8_quantize(r)                                                  # of what was just written
            done()
            fp8_block_mm(a, s, w, sw, bias=r[0, :N], out=y)                         # y over the last round's
            done()
            fp8_block_mm(a[:, :N], y[:, :4], w2, sw2, out=z)                        # y as scales, z over the last round's
            done()
            kept += [h, r.clone(), y.clone(), z.clone()]
        return kept

    want, got = chain(True), chain(False)
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.isfinite(b).any()


def test_autograd_notices_written_outputs(dev):
    """A value that autograd kept for a backward pass and that an operator then overwrites is noticed, as with torch's own
    in-place operators."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_block_mm, fp8_quantize
    from qwen_a100_fastpath_b200.norms import residual_norm
    leaf = torch.ones(4, 256, device=dev, requires_grad=True)
    x = torch.ones(4, 256, device=dev, dtype=torch.bfloat16)
    a, sa = fp8_quantize(x)
    w = torch.ones(256, 256, device=dev).to(torch.float8_e4m3fn).t()
    for write in (lambda r: residual_norm(x, r, x[0], residual_out=r),
                  lambda r: fp8_block_mm(a, sa, w, torch.ones(2, 2, device=dev), out=r)):
        kept = leaf.exp()                              # its backward needs the value itself
        write(kept.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.sum().backward()
        with pytest.raises(ValueError, match="requires a gradient"):
            write(leaf.exp())
        with pytest.raises(ValueError, match="requires a gradient"):
            write(leaf)
    assert (leaf == 1).all()
