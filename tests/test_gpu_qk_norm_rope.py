"""Norms of queries and keys for each head with the rotation (norms.qk_norm_rope) against float64.

Tolerance: a row's mean of squares is an fp32 sum of at most D / 32 + 5 terms a lane and step (D <= 512: 21 roundings), the
product with 1 / D, the addition, the reciprocal root (2 units) and its product with the weight are five more, half of what
comes under the root; the product with x and the two of the rotation, with its sum, another four: at most 24 units of 2^-24
of |a cos| + |b sin|.  The result is rounded once: 2^-8 of it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as orc
from tests.test_gpu_kv4 import check_written, host, random_cache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def table(dev, n, rot, dtype=torch.float32):
    angle = torch.arange(n, device=dev, dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / max(rot, 1))
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype)


def check(got, x, weight, positions, cos_sin, eps, offset, interleaved):
    ref, size = orc.norm_rope(host(x), None if weight is None else host(weight), host(positions),
                              None if cos_sin is None else host(cos_sin), eps, offset, interleaved)
    got = host(got)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    err, bound = np.abs(got - ref), 2.0 ** -8 * np.abs(ref) * (1 + 2.0 ** -7) + 24 * 2.0 ** -24 * size + 2.0 ** -134
    ok = np.isnan(ref) | (err <= bound)
    assert ok.all(), (np.argwhere(~ok)[:4], np.nanmax(err / bound))


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (80, 80), (96, 24), (128, 128), (128, 20), (192, 64), (256, 64),
                                   (256, 256), (512, 128), (40, 0), (17, 16), (1, 0), (2, 2), (511, 510)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_and_rotations(dev, d, rot, interleaved):
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(d + rot)
    T, h, hkv = 37, 5, 2
    q = (3 * torch.randn(T, h, d, device=dev, generator=gen)).to(BF16)
    k = torch.randn(T, hkv, d, device=dev, generator=gen).to(BF16)
    qw, kw = (1 + 0.3 * torch.randn(2, d, device=dev, generator=gen)).to(BF16)
    pos = torch.randint(0, 5000, (T,), device=dev, generator=gen)
    cs = table(dev, 5000, rot) if rot else None
    a, b = qk_norm_rope(q, k, qw, kw, pos, cs, eps=1e-5, interleaved=interleaved)
    check(a, q, qw, pos, cs, 1e-5, 0.0, interleaved)
    check(b, k, kw, pos, cs, 1e-5, 0.0, interleaved)


@pytest.mark.parametrize("T,h,hkv", [(1, 1, 1), (1, 24, 4), (5, 24, 4), (1000, 3, 1), (64, 0, 2), (64, 2, 0), (0, 4, 2)])
@pytest.mark.parametrize("d", [128, 256])
def test_tokens_and_counts(dev, d, T, h, hkv):
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(T)
    q, k = (torch.randn(T, n, d, device=dev, generator=gen).to(BF16) for n in (h, hkv))
    qw, kw = (0.3 * torch.randn(2, d, device=dev, generator=gen)).to(BF16)
    pos = torch.randint(0, 300, (T,), device=dev, generator=gen)
    cs = table(dev, 300, 64, BF16)
    a, b = qk_norm_rope(q, k, qw, kw, pos, cs, weight_offset=1.0)
    assert a.shape == q.shape and b.shape == k.shape and a.is_contiguous() and b.is_contiguous()
    check(a, q, qw, pos, cs, 1e-6, 1.0, False)
    check(b, k, kw, pos, cs, 1e-6, 1.0, False)


@pytest.mark.parametrize("weights", [(False, False), (True, False), (False, True)])
def test_without_norms(dev, weights):
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(1)
    q, k = (torch.randn(19, n, 128, device=dev, generator=gen).to(BF16) for n in (6, 2))
    qw, kw = (torch.randn(128, device=dev, generator=gen).to(BF16) if w else None for w in weights)
    pos = torch.arange(19, device=dev)
    cs = table(dev, 19, 128)
    a, b = qk_norm_rope(q, k, qw, kw, pos, cs)
    check(a, q, qw, pos, cs, 1e-6, 0.0, False)
    check(b, k, kw, pos, cs, 1e-6, 0.0, False)
    a, b = qk_norm_rope(q, k, None, None, None, None)    # neither norm nor rotation: a copy
    assert torch.equal(a, q) and torch.equal(b, k)


def test_strides_and_edges(dev):
    """Views of the qkv product (with a gate between the query's heads), broadcast and transposed inputs, odd addresses;
    positions outside the table; rows of zeros, of infinities, of very large and very small values."""
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(2)
    T, d = 12, 128
    rows = torch.randn(T, 6 * 2 * d + 4 * d, device=dev, generator=gen).to(BF16)
    gated = rows[:, :6 * 2 * d].unflatten(1, (6, 2 * d))[..., :d]
    kv = rows[:, 6 * 2 * d:].unflatten(1, (4, d))
    qw, kw = (1 + 0.3 * torch.randn(2, 2 * d, device=dev, generator=gen)).to(BF16)[:, ::2]
    pos = torch.tensor([0, 5, -1, 99, 100, 2 ** 40, -2 ** 50, 7, 8, 9, 10, 11], device=dev)
    cs = table(dev, 200, 96)[::2]
    odd = torch.randn(T, 6, d + 1, device=dev, generator=gen).to(BF16)[..., 1:]
    for q, k in ((gated, kv[:, :2]), (odd, kv[:, 3:4].expand(T, 2, d)),
                 (torch.randn(6, T, d, device=dev, generator=gen).to(BF16).transpose(0, 1), kv[:, ::3]),
                 (torch.randn(d, T, 6, device=dev, generator=gen).to(BF16).permute(1, 2, 0), kv[:1].expand(T, 4, d))):
        a, b = qk_norm_rope(q, k, qw, kw, pos, cs)
        check(a, q, qw, pos, cs, 1e-6, 0.0, False)
        check(b, k, kw, pos, cs, 1e-6, 0.0, False)
        assert a[:, :, :96].isnan().any(2).any(1).tolist() == [p < 0 or p >= 100 for p in pos.tolist()]
        assert not a[:, :, 96:].isnan().any()
    x = torch.randn(6, 1, d, device=dev, generator=gen)
    x[0] = 0
    x[1] *= 1e18
    x[2] *= 1e-25
    x[3, 0, 100] = float("nan")
    x = x.to(BF16)
    pos = torch.arange(6, device=dev)
    a, _ = qk_norm_rope(x, x, qw, kw, pos, cs)
    check(a, x, qw, pos, cs, 1e-6, 0.0, False)
    assert not a[0].any() and a[3].isnan().all()


@pytest.mark.parametrize("d,rot", [(128, 64), (256, 64), (64, 0), (96, 20)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_an_infinite_weight_of_values_that_do_not_turn(dev, d, rot, interleaved):
    """It makes them infinite, in every form of the kernel, and leaves the others as they are."""
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(d)
    q = (2 + torch.rand(9, 6, d, device=dev, generator=gen)).to(BF16) * torch.tensor([1, -1] * 3, device=dev)[:, None]
    q = q.to(BF16)
    w = (1 + 0.3 * torch.randn(d, device=dev, generator=gen)).to(BF16)
    pos, cs = torch.arange(9, device=dev), table(dev, 9, rot) if rot else None
    a, b = qk_norm_rope(q, q, w, w, pos, cs, interleaved=interleaved)
    at = torch.zeros(d, dtype=torch.bool, device=dev)
    at[[rot + 3, d - 1]] = True
    w[at] = float("inf")
    x, y = qk_norm_rope(q, q, w, w, pos, cs, interleaved=interleaved)
    for got, ref in ((x, a), (y, b)):
        assert torch.equal(got[..., ~at], ref[..., ~at])
        assert torch.equal(got[..., at].float(), torch.sign(q[..., at].float()) * float("inf"))


def test_a_table_of_no_positions(dev):
    """Every position is outside it."""
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    x = torch.ones(3, 2, 128, device=dev, dtype=BF16)
    a, b = qk_norm_rope(x, x, None, None, torch.arange(3, device=dev), torch.empty(0, 64, device=dev))
    for t in (a, b):
        assert t[..., :64].isnan().all() and torch.equal(t[..., 64:], x[..., 64:])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("T,h,hkv,rot,interleaved", [(3000, 16, 2, 64, False), (1, 4, 1, 64, False), (5, 24, 4, 32, False), (133, 3, 3, 20, True),
                                                     (40, 0, 2, 64, False), (64, 8, 8, 0, False)])
def test_into_the_cache(dev, d, T, h, hkv, rot, interleaved):
    """The same bits as the two calls that it replaces."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(T + d)
    page = 16
    pages = max(20, T // page + 1)
    cache = random_cache(gen, pages, page, hkv, d)
    before = KV4Cache(*(t.clone() for t in cache))
    qkv = torch.randn(T, h + 2 * hkv, d, device=dev, generator=gen).to(BF16)
    q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    kw = (1 + 0.3 * torch.randn(d, device=dev, generator=gen)).to(BF16)
    pos = torch.randint(0, 100, (T,), device=dev, generator=gen)
    cs = table(dev, 100, rot) if rot else None
    slots = torch.randperm(pages * page, generator=gen, device=dev)[:T]
    if T > 3:
        slots[2], slots[3], pos[1] = -1, pages * page, 100
    a, none = qk_norm_rope(q, k, kw, kw, pos, cs, interleaved=interleaved, v=v, cache=cache, slots=slots)
    b, kr = qk_norm_rope(q, k, kw, kw, pos, cs, interleaved=interleaved)
    assert none is None and torch.equal(a.nan_to_num(7), b.nan_to_num(7))
    check_written(cache, before, kr, v, slots)


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (80, 80), (128, 128), (192, 64), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_rows(dev, d, rot, interleaved):
    """On both sides of the number of rows from which several heads share a group of lanes, with head counts that do not fill
    the last group, against float64; and the same bits into the cache."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(d + rot)
    h, hkv, page = 12, 3, 16
    lanes = 8 if d <= 64 else 16 if d <= 128 else 32
    rows = (1 << 17) // lanes * 8
    qw, kw = (0.3 * torch.randn(2, d, device=dev, generator=gen)).to(BF16)
    cs = table(dev, 500, rot)
    for T in (rows // (h + hkv) - 1, rows // (h + hkv) + 3):
        qkv = torch.randn(T, h + 2 * hkv, d, device=dev, generator=gen).to(BF16)
        q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        pos = torch.randint(0, 500, (T,), device=dev, generator=gen)
        a, b = qk_norm_rope(q, k, qw, kw, pos, cs, weight_offset=1.0, interleaved=interleaved)
        check(a, q, qw, pos, cs, 1e-6, 1.0, interleaved)
        check(b, k, kw, pos, cs, 1e-6, 1.0, interleaved)
    if d in (64, 128, 256):
        pages = T // page + 1
        cache = random_cache(gen, pages, page, hkv, d)
        before = KV4Cache(*(t.clone() for t in cache))
        slots = torch.randperm(pages * page, generator=gen, device=dev)[:T]
        slots[5], slots[T - 2] = -1, pages * page
        c, _ = qk_norm_rope(q, k, qw, kw, pos, cs, weight_offset=1.0, interleaved=interleaved, v=v, cache=cache, slots=slots)
        assert torch.equal(c, a)
        check_written(cache, before, b, v, slots)


def test_two_streams_and_a_graph(dev):
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(8)
    q, k = (torch.randn(300, n, 256, device=dev, generator=gen).to(BF16) for n in (24, 4))
    w = torch.ones(256, device=dev, dtype=BF16)
    pos, cs = torch.arange(300, device=dev), table(dev, 300, 64)
    first = qk_norm_rope(q, k, w, w, pos, cs)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = qk_norm_rope(q, k, w, w, pos, cs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = qk_norm_rope(q, k, w, w, pos, cs)
    q.mul_(2)
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, caught):
        assert torch.equal(a, b) and torch.equal(a, c)
