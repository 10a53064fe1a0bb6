"""The residual update with the norms on both sides of a block (norms.py over qf_residual_norm) against the float64
oracle, and the decoder layer's linear path of norms.py and fp8.py together.

Tolerances, in units of u = 2^-24.  A mean of squares of H <= 16384 terms summed in a tree: each term squared (1), at
most 32 in a thread's chain, 5 shuffles, 16 warps, the division and eps: under 60 u, halved by the square root; rsqrt
itself 4 u: a norm factor is good to 36 u, a normed value to 40 u.  An activation: exp 4 u (its argument is exact), sum
and quotient: 8 u.  So v = alpha * u * act(gate) is good to 52 u of itself and r to 52 u of |v| plus 1 u of |r|.  h is
built from r: 40 u of itself, plus the error of r, times the norm factor, plus a factor's change by r's errors in the
mean (at most 52 u where |v| dominates, taken of h).  Stored results add half a step of their type.
"""
from __future__ import annotations

import itertools

import numpy as np
import pytest

from oracle import fp8_oracle as orc
from tests.test_gpu_fp8 import check_mm, f64, make_weight

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def bf16(dev, a):
    import torch
    return torch.from_numpy(np.asarray(a, np.float32)).to(dev).to(torch.bfloat16)


def make(dev, M, H, gate="full", residual="bf16", seed=0):
    import torch
    rs = np.random.RandomState(seed)
    x = bf16(dev, rs.standard_normal((M, H)))
    r = bf16(dev, 2 * rs.standard_normal((M, H)))
    if residual == "f32":
        r = r.float() + torch.from_numpy(rs.standard_normal((M, H)).astype(np.float32) * 1e-3).to(dev)
    shape = {"none": None, "full": (M, H), "channel": (H,), "token": (M, 1), "row": (1, H), "one": (1,)}[gate]
    g = None if shape is None else bf16(dev, 2 * rs.standard_normal(shape))
    return x, r, g, bf16(dev, 1 + 0.2 * rs.standard_normal(H)), bf16(dev, 1 + 0.2 * rs.standard_normal(H))


def check(h, r_got, x, r, pre, post, g, act, alpha, offset, quantize):
    import torch
    n = lambda t: None if t is None else f64(t)  # noqa: E731
    gg = None if g is None else np.broadcast_to(f64(g), x.shape)
    h_o, r_o, v_o = orc.residual_norm(f64(x), n(r), n(pre), EPS, n(post), gg, act, alpha, offset)
    half = 2.0 ** -24 if r_got.dtype == torch.float32 else 2.0 ** -8
    e_r = 52 * U * np.abs(v_o) + U * np.abs(r_o)
    err = np.abs(f64(r_got) - r_o)
    assert np.all(err <= half * np.abs(r_o) + (1 + half) * e_r + 1e-38), np.max(err / (half * np.abs(r_o) + e_r + 1e-38))
    if pre is None:
        assert h is None
        return
    # the norm factor with its weight, dh/dr (|h| / |r| is not defined where r cancels to zero: 1.75 - 0.7 * 2.5)
    factor = np.abs(f64(pre) + offset)[None, :] / np.sqrt(np.mean(r_o * r_o, axis=1, keepdims=True) + EPS)
    e_h = 92 * U * np.abs(h_o) + factor * e_r
    if not quantize:
        err = np.abs(f64(h) - h_o)
        assert np.all(err <= 2.0 ** -8 * np.abs(h_o) + 1.01 * e_h + 1e-38), np.max(err / (2.0 ** -8 * np.abs(h_o) + e_h + 1e-38))
        return
    q, s = h
    assert q.dtype == torch.float8_e4m3fn
    for c0 in range(0, x.shape[1], 128):
        c = slice(c0, min(x.shape[1], c0 + 128))
        top = np.maximum(np.abs(h_o[:, c]).max(axis=1), 448 * 2.0 ** -60)
        e_top = e_h[:, c].max(axis=1) + 4 * U * top
        got_s = f64(s)[:, c0 // 128]
        assert np.all(np.abs(got_s - top / 448) <= e_top / 448)
        err = np.abs(f64(q)[:, c] * got_s[:, None] - h_o[:, c])
        # half a step of the value, or of the values below 2^-6; the scale's own error moves a value by its part of it
        tol = np.maximum(2.0 ** -4 * np.abs(h_o[:, c]), 2.0 ** -10 * got_s[:, None]) * (1 + 2.0 ** -10) + \
            2 * e_h[:, c] + np.abs(h_o[:, c]) * (2 * e_top / top)[:, None]
        assert np.all(err <= tol), np.max(err / tol)


@pytest.mark.parametrize("residual,quantize,post,gate,act", [
    c for c in itertools.product(("bf16", "f32"), (False, True), (False, True), ("none", "full", "channel", "token"),
                                 ("none", "sigmoid", "silu")) if c[3] != "none" or c[4] == "none"])
def test_options(dev, residual, quantize, post, gate, act):
    from qwen_a100_fastpath_b200.norms import residual_norm
    x, r, g, pre, pw = make(dev, 5, 1160, gate, residual, seed=7)
    pw = pw if post else None
    h, ro = residual_norm(x, r, pre, eps=EPS, post_weight=pw, gate=g, gate_act=act, residual_scale=0.7, weight_offset=0.5,
                          quantize=quantize)
    assert ro.dtype == r.dtype and ro.shape == r.shape
    check(h, ro, x, r, pre, pw, g, act, 0.7, 0.5, quantize)


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("M,H", [(1, 1), (1, 7), (2, 8), (1, 128), (3, 129), (4, 255), (1, 5120), (2, 4096), (3, 4104), (2, 8192),
                                 (2, 8200), (1, 16384), (3, 16383), (3000, 136), (1201, 5120), (5000, 8), (2500, 2568), (900, 8192), (700, 16384)])
def test_sizes(dev, M, H, quantize):
    from qwen_a100_fastpath_b200.norms import residual_norm
    x, r, g, pre, pw = make(dev, M, H, "full", "f32", seed=M + H)
    h, ro = residual_norm(x, r, pre, eps=EPS, post_weight=pw, gate=g, gate_act="silu", quantize=quantize)
    check(h, ro, x, r, pre, pw, g, "silu", 1.0, 0.0, quantize)


@pytest.mark.parametrize("H", [512, 520, 333])
def test_strides_in_place_and_optional_parts(dev, H):
    """Rows of other strides and alignments, the residual updated in place, neighbours left as they were, a call without
    a residual and one without the second norm; the same bits whatever the layout."""
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    M = 6
    x, r, g, pre, pw = make(dev, M, H, "full", "bf16", seed=H)
    kw = dict(eps=EPS, post_weight=pw, gate_act="sigmoid", residual_scale=0.5)
    h, ro = residual_norm(x, r, pre, gate=g, **kw)
    check(h, ro, x, r, pre, pw, g, "sigmoid", 0.5, 0.0, False)

    def strided(t, pad, off):
        buf = torch.full((M, H + pad + off), 9.0, dtype=t.dtype, device=dev)
        v = buf[:, off:off + H]
        v.copy_(t)
        return buf, v

    for pad, off in ((8, 8), (3, 1)):
        (_, x2), (rb, r2), (_, g2) = strided(x, pad, off), strided(r, pad, off), strided(g, pad, off)
        h2, r3 = residual_norm(x2, r2, pre, gate=g2, residual_out=r2, **kw)
        assert r3 is r2 and torch.equal(h2, h) and torch.equal(r2, ro)
        r2.fill_(9.0)
        assert (rb == 9.0).all()
    h3, r4 = residual_norm(x.view(2, 3, H), r.view(2, 3, H), pre, gate=g.view(2, 3, H), **kw)
    assert h3.shape == (2, 3, H) and torch.equal(h3.view(M, H), h) and torch.equal(r4.view(M, H), ro)
    h4, r5 = residual_norm(x, None, pre, gate=g, **kw)
    check(h4, r5, x, None, pre, pw, g, "sigmoid", 0.5, 0.0, False)
    h5, r6 = residual_norm(x, r, None, gate=g, **kw)
    assert h5 is None and torch.equal(r6, ro)
    for gate in ("row", "one"):
        gb = make(dev, M, H, gate, seed=H)[2]
        hb, rb2 = residual_norm(x, r, pre, gate=gb, **kw)
        check(hb, rb2, x, r, pre, pw, gb, "sigmoid", 0.5, 0.0, False)
    h0, r0 = residual_norm(x[:0], r[:0], pre, quantize=True)
    assert h0[0].shape == (0, H) and r0.shape == (0, H)


@pytest.mark.parametrize("residual", ["bf16", "f32"])
@pytest.mark.parametrize("gate", ["none", "full", "channel", "token"])
def test_many_rows_in_place(dev, residual, gate):
    """Several rows to a CTA (they arrive ahead in shared memory): every kind of gate, the residual updated in place with
    neighbours left as they were, the same bits as calls of a few rows."""
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    M, H = 2600, 1024
    x, r, g, pre, pw = make(dev, M, H, gate, residual, seed=11)
    kw = dict(eps=EPS, post_weight=pw, gate_act="sigmoid" if gate != "none" else "none", residual_scale=0.7)
    parts = [slice(0, 7), slice(1300, 1310), slice(M - 5, M)]
    few = [residual_norm(x[p], r[p], pre, gate=g[p] if gate in ("full", "token") else g, **kw) for p in parts]
    buf = torch.full((M + 2, H + 8), 9.0, dtype=r.dtype, device=dev)
    r2 = buf[1:M + 1, :H]
    r2.copy_(r)
    h, ro = residual_norm(x, r2, pre, gate=g, residual_out=r2, **kw)
    assert ro is r2
    for p, (hf, rf) in zip(parts, few):
        assert torch.equal(h[p], hf) and torch.equal(r2[p], rf)
    check(h, r2, x, r, pre, pw, g, kw["gate_act"], 0.7, 0.0, False)
    assert residual_norm(x, r, None, gate=g, **kw)[0] is None
    assert torch.equal(residual_norm(x, r, None, gate=g, **kw)[1], r2)
    r2.fill_(9.0)
    assert (buf == 9.0).all()


@pytest.mark.parametrize("quantize", [False, True])
def test_special_rows(dev, quantize):
    """A row of zeros gives zeros; what is not finite stays in its own row; large values do not overflow the sum."""
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    x, r, _, pre, pw = make(dev, 6, 640, "none", "f32", seed=3)
    base, rb = residual_norm(x, r, pre, eps=EPS, quantize=quantize)
    x[1], r[1] = 0.0, 0.0
    x[2, 5] = float("nan")
    r[3, 600] = float("inf")
    x[4], r[4] = x[4] * 1e15, 0.0
    h, ro = residual_norm(x, r, pre, eps=EPS, quantize=quantize)
    q = f64(h[0] if quantize else h)
    assert not q[1].any() and np.isnan(q[2]).any() and np.isfinite(q[4]).all() and torch.isinf(ro[3, 600])
    b = f64(base[0] if quantize else base)
    assert np.array_equal(q[[0, 5]], b[[0, 5]]) and torch.equal(ro[[0, 5]], rb[[0, 5]])
    if quantize:
        assert torch.equal(h[1][1], torch.full_like(h[1][1], 2.0 ** -60)) and torch.isnan(h[1][2]).all()


def test_refusals(dev):
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    x, r, g, pre, pw = make(dev, 4, 256)
    cases = [
        lambda: residual_norm(x.float(), r, pre), lambda: residual_norm(x, r[:3], pre), lambda: residual_norm(x, r.half(), pre),
        lambda: residual_norm(x, r, pre[:255]), lambda: residual_norm(x, r, pre.float()), lambda: residual_norm(x, r.cpu(), pre),
        lambda: residual_norm(x, r, None, quantize=True), lambda: residual_norm(x, r, pre, gate_act="silu"),
        lambda: residual_norm(x, r, pre, gate=g[:, :100]), lambda: residual_norm(x, r, pre, gate=g[None]),
        lambda: residual_norm(x, r, pre, eps=-1.0), lambda: residual_norm(x, r, pre, eps=float("nan")),
        lambda: residual_norm(x, r, pre, residual_out=r.float()), lambda: residual_norm(x, r, pre, residual_out=r[:3]),
        lambda: residual_norm(x, r, pre, residual_out=torch.empty(256, 4, device=dev, dtype=torch.bfloat16).t()),
        lambda: residual_norm(x.clone().requires_grad_(), r, pre),
        lambda: residual_norm(torch.zeros(1, 16385, device=dev, dtype=torch.bfloat16), None, None),
    ]
    for i, f in enumerate(cases):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was taken")
    buf = torch.zeros(5 * 256, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="single memory location"):
        residual_norm(x, buf[:1024].view(4, 256), pre, residual_out=buf[256:].view(4, 256))
    with pytest.raises(RuntimeError, match="single memory location"):
        residual_norm(x, r, pre, residual_out=x)
    torch.cuda.synchronize(dev)


# ---- the layer ---------------------------------------------------------------------------------------------------
class Layer:
    """Linear path of a decoder layer on block-scaled fp8 weights: norm -> qkv -> (attention: its output taken as a slice
    of qkv) -> o_proj -> norm -> gate_up -> silu gate -> down -> norm of the next layer."""

    def __init__(self, dev, hidden=512, inner=1280):
        self.qkv, self.o = make_weight(dev, 1024, hidden, 1), make_weight(dev, hidden, 640, 2)
        self.gate_up, self.down = make_weight(dev, 2 * inner, hidden, 3), make_weight(dev, hidden, inner, 4)
        rs = np.random.RandomState(5)
        self.norm = [bf16(dev, 1 + 0.1 * rs.standard_normal(hidden)) for _ in range(3)]

    def __call__(self, x, residual):
        from qwen_a100_fastpath_b200.fp8 import fp8_block_linear, fp8_block_mm, fp8_quantize
        from qwen_a100_fastpath_b200.norms import residual_norm
        (q, s), residual = residual_norm(x, residual, self.norm[0], quantize=True)
        att = fp8_block_mm(q, s, *self.qkv[:2])[:, :640]
        x = fp8_block_linear(att, *self.o[:2])
        (q, s), residual = residual_norm(x, residual, self.norm[1], quantize=True)
        gu = fp8_block_mm(q, s, *self.gate_up[:2])
        x = fp8_block_mm(*fp8_quantize(gu, silu_mul=True), *self.down[:2])
        return residual_norm(x, residual, self.norm[2])

    def stepwise(self, x, residual):
        """The same layer checked operator by operator: each one's float64 value from the inputs it was given."""
        from qwen_a100_fastpath_b200.fp8 import fp8_block_linear, fp8_block_mm, fp8_quantize
        from qwen_a100_fastpath_b200.norms import residual_norm

        def mm(q, s, w):
            y = fp8_block_mm(q, s, *w[:2])
            check_mm(y, *orc.block_mm(f64(q), f64(s), w[2], f64(w[1])), q.shape[1])
            return y

        def norm(x, r, w, quantize):
            h, ro = residual_norm(x, r, w, eps=EPS, quantize=quantize)
            check(h, ro, x, r, w, None, None, "none", 1.0, 0.0, quantize)
            return h, ro

        (q, s), residual = norm(x, residual, self.norm[0], True)
        att = mm(q, s, self.qkv)[:, :640]
        x = fp8_block_linear(att, *self.o[:2])
        check_mm(x, *orc.block_mm(*orc.quantize(f64(att)), self.o[2], f64(self.o[1])), 640)
        (q, s), residual = norm(x, residual, self.norm[1], True)
        x = mm(*fp8_quantize(mm(q, s, self.gate_up), silu_mul=True), self.down)
        return norm(x, residual, self.norm[2], False)


@pytest.mark.parametrize("M", [1, 5, 16, 40, 300])
def test_layer(dev, M):
    """The operators together: eager, captured and replayed on new inputs, and on two streams at once."""
    import torch
    layer = Layer(dev)
    rs = np.random.RandomState(M)

    def inputs():
        return bf16(dev, rs.standard_normal((M, 512))), torch.from_numpy(rs.standard_normal((M, 512)).astype(np.float32)).to(dev)

    x, r = inputs()
    h, ro = layer(x, r)
    h2, ro2 = layer.stepwise(x, r)
    assert torch.equal(h, h2) and torch.equal(ro, ro2)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    sx, sr = x.clone(), r.clone()
    graphs = []
    for _ in range(2):                                  # two graphs of the same calls
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            graphs.append((g, layer(sx, sr)))
    for k in range(3):
        x, r = inputs()
        want = layer(x, r)
        sx.copy_(x)
        sr.copy_(r)
        g, got = graphs[k % 2]
        g.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # two streams at once, each with its own inputs
    pairs = [inputs() for _ in range(2)]
    want = [layer(*p) for p in pairs]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize(dev)
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = layer(*pairs[i])
    torch.cuda.synchronize(dev)
    for i in range(2):
        assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
