"""The block-scaled fp8 operators and the residual norm under tracing (no device): a symbolic token count stays symbolic, and
types and shapes that a real call refuses are refused there too."""
from __future__ import annotations

import pytest
import torch

from qwen_a100_fastpath_b200 import fp8, norms

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


class Layer(torch.nn.Module):
    """The linear path of a decoder layer: every operator, its optional parts and an output given."""

    def __init__(self, device="cpu", hidden=256, inner=384):
        super().__init__()
        def w(n, k):
            return torch.zeros(n, k, dtype=E4M3, device=device), torch.ones(-(-n // 128), -(-k // 128), device=device)
        self.qkv, self.o, self.gate_up, self.down = w(512, hidden), w(hidden, 500), w(2 * inner, hidden), w(hidden, inner)
        self.norm = torch.ones(hidden, dtype=BF16, device=device)
        self.bias = torch.zeros(512, dtype=BF16, device=device)

    def forward(self, x, residual):
        (q, s), residual = norms.residual_norm(x, residual, self.norm, quantize=True)
        att = fp8.fp8_block_mm(q, s, self.qkv[0].t(), self.qkv[1], bias=self.bias)[:, :500]
        x = fp8.fp8_block_linear(att, self.o[0].t(), self.o[1])
        h, residual = norms.residual_norm(x, residual, self.norm, post_weight=self.norm, gate=x, gate_act="silu",
                                          residual_out=residual)
        gu = fp8.fp8_block_mm(*fp8.fp8_quantize(h), self.gate_up[0].t(), self.gate_up[1])
        a, s = fp8.fp8_quantize(gu, silu_mul=True)
        y = fp8.fp8_block_mm(a, s, self.down[0].t(), self.down[1], out=torch.empty_like(residual))
        return y, residual


def inputs(tokens, device="cpu"):
    return torch.zeros(tokens, 256, dtype=BF16, device=device), torch.zeros(tokens, 256, device=device)


def test_make_fx_keeps_the_token_count():
    from torch.fx.experimental.proxy_tensor import make_fx
    layer = Layer()
    gm = make_fx(lambda x, r: layer(x, r), tracing_mode="symbolic", _allow_non_fake_inputs=True)(*inputs(7))
    calls = [n for n in gm.graph.nodes if n.op == "call_function" and "qf_b200" in str(n.target)]
    assert len(calls) == 8
    seen = 0
    for n in calls:
        val = n.meta.get("val")
        for v in val if isinstance(val, (tuple, list)) else (val,):
            if isinstance(v, torch.Tensor):
                seen += 1
                assert isinstance(v.shape[0], torch.SymInt) and not v.shape[0].node.expr.is_number, (n, v.shape)
    assert seen >= 11


def test_export_with_dynamic_tokens():
    tokens = torch.export.Dim("tokens")
    ep = torch.export.export(Layer(), inputs(7), dynamic_shapes=({0: tokens}, {0: tokens}))
    y = next(n for n in ep.graph.nodes if n.op == "output").args[0]
    assert all(not isinstance(v.meta["val"].shape[0], int) for v in y)


def test_int8_linear_keeps_the_token_count():
    from torch.fx.experimental.proxy_tensor import make_fx
    from qwen_a100_fastpath_b200._lib import load_torch_ops
    op = load_torch_ops()
    w, s = torch.zeros(64, 256, dtype=torch.int8).t(), torch.ones(64)
    trace = make_fx(lambda x: op(x, w, s, None), tracing_mode="symbolic", _allow_non_fake_inputs=True)
    gm = trace(torch.zeros(7, 256, dtype=BF16))
    out = next(n for n in gm.graph.nodes if "int8_linear" in str(n.target)).meta["val"]
    assert isinstance(out.shape[0], torch.SymInt) and not out.shape[0].node.expr.is_number and out.shape[1] == 64


@pytest.mark.parametrize("shape", [(256,), (5, 256), (2, 3, 256), (2, 0, 130), (4, 1001)])
def test_results_have_the_layout_of_a_contiguous_call(shape):
    x = torch.empty(shape, dtype=BF16, device="meta")
    q, s = fp8.fp8_quantize(x)
    kp = -(-shape[-1] // 16) * 16
    assert q.shape == x.shape and q.stride() == torch.empty(*shape[:-1], kp, device="meta").stride()
    assert s.shape == (*shape[:-1], -(-shape[-1] // 128)) and s.is_contiguous()


def test_refusals_of_types_and_shapes():
    m = "meta"
    x, r = torch.empty(4, 256, dtype=BF16, device=m), torch.empty(4, 256, device=m)
    a, sa = fp8.fp8_quantize(x)
    w, sw = torch.empty(300, 256, dtype=E4M3, device=m).t(), torch.empty(3, 2, device=m)
    n = torch.empty(256, dtype=BF16, device=m)
    fp8.fp8_block_mm(a, sa, w, sw)
    norms.residual_norm(x, r, n)
    cases = [
        lambda: fp8.fp8_quantize(x.float()), lambda: fp8.fp8_quantize(x[:, :255], silu_mul=True),
        lambda: fp8.fp8_block_mm(a, sa, w, torch.empty(9, 9, device=m)), lambda: fp8.fp8_block_mm(a, sa[:3], w, sw),
        lambda: fp8.fp8_block_mm(a, sa.double(), w, sw), lambda: fp8.fp8_block_mm(a[0], sa[0], w, sw),
        lambda: fp8.fp8_block_mm(a, sa, w[:128], sw), lambda: fp8.fp8_block_mm(a, sa, w, sw, bias=n),
        lambda: fp8.fp8_block_mm(a, sa, w, sw, out=torch.empty(4, 301, device=m)),
        lambda: fp8.fp8_block_mm(a, sa, w, sw, out=torch.empty(4, 300, device=m, dtype=torch.float16)),
        lambda: fp8.fp8_block_linear(x[:, :128], w, sw), lambda: fp8.fp8_block_linear(r, w, sw),
        lambda: norms.residual_norm(x, r[:3], n), lambda: norms.residual_norm(x, r.half(), n),
        lambda: norms.residual_norm(x, r, n[:100]), lambda: norms.residual_norm(x, r, None, quantize=True),
        lambda: norms.residual_norm(x, r, n, gate=x[:, :100]), lambda: norms.residual_norm(x, r, n, gate=x[None]),
        lambda: norms.residual_norm(x, r, n, gate_act="silu"), lambda: norms.residual_norm(x, r, n, residual_out=x),
        lambda: norms.residual_norm(x, r, n, residual_out=r[:2]), lambda: norms.residual_norm(x, r, n, eps=-1.0),
    ]
    for i, f in enumerate(cases):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was taken")


def test_written_outputs_raise_their_version():
    m = "meta"
    x, r = torch.empty(4, 256, dtype=BF16, device=m), torch.empty(4, 256, device=m)
    norms.residual_norm(x, r, None, residual_out=r)
    assert r._version == 1 and r[:2]._version == 1
    a, sa = fp8.fp8_quantize(x)
    out = torch.empty(8, 300, device=m)
    fp8.fp8_block_mm(a, sa, torch.empty(300, 256, dtype=E4M3, device=m).t(), torch.empty(3, 2, device=m), out=out[2:6])
    assert out._version == 1 and a._version == 0 and x._version == 0


def test_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    m = "meta"
    x, n = torch.empty(4, 256, dtype=BF16, device=m), torch.empty(256, dtype=BF16, device=m)
    r = torch.empty(4, 256, device=m)
    a, sa = fp8.fp8_quantize(x)
    w, sw = torch.empty(300, 256, dtype=E4M3, device=m).t(), torch.empty(3, 2, device=m)
    leaf = n.clone().requires_grad_()
    out = torch.empty(4, 300, device=m, requires_grad=True)
    with pytest.raises(ValueError, match="requires a gradient"):
        norms.residual_norm(x, r, leaf)
    for t in (out, out * 1):
        with pytest.raises(ValueError, match="out requires a gradient"):
            fp8.fp8_block_mm(a, sa, w, sw, out=t)
    with torch.no_grad():
        norms.residual_norm(x, r, leaf)
        fp8.fp8_block_mm(a, sa, w, sw, out=out)
    with torch.inference_mode():
        norms.residual_norm(x, r, leaf, residual_out=torch.empty(4, 256, device=m))
    kept = torch.inference_mode()(lambda: torch.empty(4, 256, device=m))()
    norms.residual_norm(x, r, n, residual_out=kept)              # an inference tensor has no version
    with fwd.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            fp8.fp8_quantize(fwd.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="tangent"):
            norms.residual_norm(x, fwd.make_dual(r, torch.ones_like(r)), n)
    f = lambda t: fp8.fp8_quantize(t)[1].sum()  # noqa: E731
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(ValueError, match="requires a gradient"):
        torch.func.grad(f)(x)
