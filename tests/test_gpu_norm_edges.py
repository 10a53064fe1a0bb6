"""The residual norm (norms.py over qf_residual_norm) at the edges of its sizes, waits and arguments."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def test_more_rows_than_2_to_the_30(dev):
    """One CTA per row and more than 2^30 of them: the row index plus the grid passes 32 bits.  Without a residual, a gate
    and a norm the result is the input."""
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    M = 2 ** 30 + 1
    x = torch.arange(M, device=dev, dtype=torch.int32).remainder_(251).to(torch.bfloat16).view(M, 1)
    buf = torch.full((M + 128, 1), 9.0, device=dev, dtype=torch.bfloat16)
    out = buf[64:M + 64]
    h, r = residual_norm(x, None, None, residual_out=out)
    assert h is None and r is out and torch.equal(out, x)
    assert (buf[:64] == 9.0).all() and (buf[M + 64:] == 9.0).all()
