"""The residual norm (norms.py over qf_residual_norm) at the edges of its sizes, waits and arguments."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

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


def ahead_against_few_rows():
    """Calls of many rows, which arrive ahead in shared memory, against calls of so few that nothing is read ahead: the same
    bits.  One, two and four pieces a thread, two to four rows in the ring, last rounds that are not full.  Returns whether a
    wait ran out in any of them."""
    import itertools

    import torch
    from qwen_a100_fastpath_b200 import _lib
    from qwen_a100_fastpath_b200.norms import residual_norm, residual_norm_status
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(5)

    def rand(*shape):
        return torch.randn(*shape, device=dev, generator=gen).to(torch.bfloat16)

    def bits(t):
        return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t

    late = False
    assert residual_norm_status(dev) == 0
    for (M, H), f32, gate, quantize in itertools.product(((3000, 1024), (2503, 5120), (700, 16384)), (False, True),
                                                         ("none", "full", "token"), (False, True)):
        x, r, pre, post = rand(M, H), rand(M, H), rand(H), rand(H)
        r = r.float() if f32 else r
        g = {"none": None, "full": rand(M, H), "token": rand(M, 1)}[gate]
        kw = dict(post_weight=post, gate_act="none" if g is None else "silu", residual_scale=0.5, quantize=quantize)
        few = []
        for m in range(0, M, 250):
            p = slice(m, min(M, m + 250))
            h, ro = residual_norm(x[p], r[p], pre, gate=g if g is None else g[p], **kw)
            few.append([bits(t) for t in (*h, ro)] if quantize else [h, ro])
        want = [torch.cat(t) for t in zip(*few)]
        assert residual_norm_status(dev) == 0
        for _ in range(3):
            ro = r.clone()
            h, _ = residual_norm(x, ro, pre, gate=g, residual_out=ro, **kw)   # in place
            got = [bits(t) for t in (*h, ro)] if quantize else [h, ro]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (M, H, f32, gate, quantize)
        st = residual_norm_status(dev)
        assert st in (0, _lib.QF_ERR_TIMEOUT)
        late = late or st != 0
    assert residual_norm_status(dev) == 0
    return late


def test_rows_ahead(dev):
    assert not ahead_against_few_rows()


def test_rows_that_arrive_late(dev):
    """Every wait for a row that is not there at the first asking runs out (a child process with the limit set to zero
    clocks): threads leave the ring at different rows while its copies are under way, the bits stay the same, and the status
    tells."""
    env = dict(os.environ, QF_TEST_OVERRIDES="1", QF_NORM_WAIT_CLOCKS="0")
    code = "from tests.test_gpu_norm_edges import ahead_against_few_rows as f; print('late' if f() else 'in time')"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and r.stdout.split()[-1] == "late", (r.stdout, r.stderr[-2000:])
