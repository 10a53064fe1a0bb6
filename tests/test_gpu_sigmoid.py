"""The gates' sigmoid and SiLU over every bf16 value of the gate, through the operators that use them, against float64.

Bounds, in units of u = 2^-24.  The sigmoid is within 2.5 u of its value where that is a normal fp32 number and within half a
step (2^-150) below; a product with it adds one rounding, u or half a step.  With x = 1, a residual of fp32 zeros and no
second norm the residual norm's result is the activation itself.  The quantizer's values v carry a sigmoid and two
products, its scales one more rounding (the quotient by 448), and e4m3 values half a step of 2^-4 or 2^-10 of the scale."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 2.0 ** -126


def gates(dev):
    import torch
    bits = torch.arange(65536, device=dev, dtype=torch.int32).to(torch.uint16).view(torch.bfloat16)
    return bits.view(256, 256)


def sigmoid(g):
    with np.errstate(over="ignore", under="ignore"):
        return np.where(g < 0, np.exp(-np.abs(g)), 1.0) / (1.0 + np.exp(-np.abs(g)))


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_every_gate(dev, act):
    import torch
    from qwen_a100_fastpath_b200.norms import residual_norm
    g = gates(dev)
    x = torch.ones_like(g)
    _, r = residual_norm(x, torch.zeros(256, 256, device=dev), None, gate=g, gate_act=act)
    got, gg = r.double().cpu().numpy(), g.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(gg) | ((gg == -np.inf) & (act == "silu")))
    ok = np.isfinite(gg)
    s = sigmoid(gg[ok])
    e_s = np.where(s >= TINY, 2.5 * U * s, 2.0 ** -150)
    ref, tol = (s, e_s) if act == "sigmoid" else (gg[ok] * s, np.abs(gg[ok]) * e_s + U * np.abs(gg[ok]) * s + 2.0 ** -150)
    err = np.abs(got[ok] - ref)
    print(act, "largest error of a normal sigmoid:", np.max(err[s >= TINY] / np.abs(ref[s >= TINY]).clip(1e-300)) / U, "u")
    assert np.all(err <= tol), (np.max(err / tol), gg[ok][np.argmax(err / tol)])
    inf = gg == np.inf
    assert np.all(got[inf] == (1.0 if act == "sigmoid" else np.inf))
    if act == "sigmoid":
        assert np.all(got[gg == -np.inf] == 0.0)


@pytest.mark.parametrize("up", [1.0, 1e30])
def test_quantizer_keeps_closed_gates(dev, up):
    """Groups of gates from -70 to -104, whose results are small but not zero: what is left of them is kept, and a large up
    value brings them back into range."""
    import torch
    from qwen_a100_fastpath_b200.fp8 import fp8_quantize
    g = torch.linspace(-104, -70, 128, device=dev).to(torch.bfloat16).view(1, 128).repeat(8, 1)
    for i in range(8):
        g[i, i * 16:] = g[i, i * 16]               # largest results at -104, -99.7 .. -74.3
    u = torch.full_like(g, up)
    q, s = fp8_quantize(torch.cat([g, u], 1), silu_mul=True)
    gg, uu = g.double().cpu().numpy(), u.double().cpu().numpy()
    sg = sigmoid(gg)
    v = gg * sg * uu
    e_g = np.where(sg >= TINY, 2.5 * U * sg, 2.0 ** -150) * np.abs(gg) + np.maximum(U * np.abs(gg) * sg, 2.0 ** -150)
    e_v = e_g * uu * (1 + U) + U * np.abs(v)
    floor = 2.0 ** -60
    top = np.maximum(np.abs(v).max(axis=1), 448 * floor)
    e_top = np.where(np.abs(v).max(axis=1) > 448 * floor, e_v.max(axis=1), 0.0)
    got_s = s.double().cpu().numpy()[:, 0]
    assert np.all(np.abs(got_s - top / 448) <= (e_top + U * top) / 448 * (1 + U))
    err = np.abs(q.double().cpu().numpy() * got_s[:, None] - v)
    # the rounding itself, relative to what was rounded; then the errors of v and of 448 / a and its product (3 u)
    tol = np.maximum(2.0 ** -4 * (np.abs(v) + e_v), 2.0 ** -10 * got_s[:, None]) + e_v + 3 * U * np.abs(v) + \
        np.abs(v) * (e_top / top)[:, None]
    assert np.all(err <= tol * (1 + 2.0 ** -20)), np.max(err / tol)
    if up > 1.0:
        assert (q.float().abs() > 0).any()
