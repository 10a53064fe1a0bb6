"""The 4-bit paged cache on the GPU (kv4.py): writer and reader bit for bit against the definition, the attention against
float64 over the values the cache stands for.

Tolerance of the attention.  The scores are fp32 sums of D exact products: off by at most (D + 8) 2^-24 of
t = scale sum |q k|, the scaling included.  A weight is then off by the factor e^(2 x that), twice for the sum it is divided
by, plus 2^-20 for the exponentials, the rescalings and the fp32 sums over tiles, and by 2^-8 for its own rounding to bf16 in
the numerator; the result is rounded to bf16 once (2^-8 of it).  With A = sum_j w_j |v_j|:
|error| <= (2^-8 + 4 (D + 8) 2^-24 t + 2^-18) A + 2^-8 |out| (1 + 2^-7)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def host(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def random_cache(gen, pages, page, hkv, d, layout="plain"):
    from qwen_a100_fastpath_b200.kv4 import KV4Cache
    dev = gen.device
    g = d // 64
    codes = torch.randint(0, 256, (2, pages, hkv, page, d // 2), device=dev, generator=gen, dtype=torch.uint8)
    s = 0.05 + 0.4 * torch.rand(2, pages, hkv, page, g, device=dev, generator=gen)
    c = -24 * s + 0.3 * torch.randn(2, pages, hkv, page, g, device=dev, generator=gen)
    scale = torch.stack([s, c], -1).to(BF16)
    if layout == "slots_first":   # [pages, slots, heads, ...] in memory
        codes = codes.transpose(2, 3).contiguous().transpose(2, 3)
        scale = scale.transpose(2, 3).contiguous().transpose(2, 3)
    elif layout == "one_tensor":  # keys and values of a page side by side, rows wider than they need
        big = torch.zeros(pages, 2, hkv, page, d // 2 + 16, dtype=torch.uint8, device=dev)
        big[..., :d // 2] = codes.transpose(0, 1)
        codes = big.transpose(0, 1)[..., :d // 2]
        scale = scale.transpose(0, 1).contiguous().transpose(0, 1)
    return KV4Cache(codes[0], codes[1], scale[0], scale[1])


def table_for(gen, lens, page, spare=0, width=None):
    """Block table of pages in random order, entries past a request's pages pointing nowhere."""
    held = [-(-max(n, 0) // page) for n in lens]
    width = max(max(held, default=0), 1) if width is None else width
    pages = max(sum(held) + spare, 1)
    order = torch.randperm(pages, generator=gen, device=gen.device).to(torch.int32).cpu()
    t = torch.full((len(lens), width), -7, dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        h = min(h, width)
        t[b, :h] = order[at:at + h]
        at += h
    return t.to(gen.device), pages


def check_attention(got, query, cache, lens, table, q_len, scale):
    d = query.shape[2]
    ref, spread, top = orc.attention(host(query), [host(t) for t in cache], lens, host(table), q_len, scale)
    got = host(got)[:len(lens) * q_len]
    bound = (2.0 ** -8 + 4 * (d + 8) * 2.0 ** -24 * top[..., None] + 2.0 ** -18) * spread + \
        2.0 ** -8 * (1 + 2.0 ** -7) * np.abs(ref)
    same_nan = np.isnan(got) == np.isnan(ref)
    assert same_nan.all(), np.argwhere(~same_nan)[:5]
    ok = np.isnan(ref) | (np.abs(got - ref) <= bound)
    assert ok.all(), (np.argwhere(~ok)[:5], np.nanmax(np.abs(got - ref) / np.maximum(bound, 1e-30)))


def run_case(dev, seed, lens, q_len, g, hkv, d, page, layout="plain", q_scale=1.0):
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(seed)
    table, pages = table_for(gen, lens, page, spare=2)
    cache = random_cache(gen, pages, page, hkv, d, layout)
    query = (q_scale * torch.randn(len(lens) * q_len, hkv * g, d, device=dev, generator=gen)).to(BF16)
    out = kv4_attention(query, cache, torch.tensor(lens, dtype=torch.int32, device=dev), table, q_len, d ** -0.5)
    assert out.shape == query.shape and out.dtype == BF16
    check_attention(out, query, cache, lens, table, q_len, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q_len,g,hkv", [(1, 1, 1), (1, 6, 4), (1, 8, 2), (3, 6, 4), (5, 5, 1), (4, 8, 3), (5, 8, 1),
                                         (6, 8, 2), (7, 7, 1), (8, 7, 1), (8, 8, 2)])
def test_attention_rows(dev, d, q_len, g, hkv):
    """Every number of row tiles; a length inside one tile and one over several."""
    run_case(dev, 10 * q_len + g, [37, 333], q_len, g, hkv, d, 16)


@pytest.mark.parametrize("page", [1, 7, 16, 64, 130, 800])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_pages_and_lengths(dev, d, page):
    """Pages that end inside a tile; lengths at and around the tiles' edges, zero and shorter than the query."""
    lens = [0, 1, 2, 3, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 255, 257, 511, 1025, 801, -3]
    run_case(dev, page, lens, 3, 2, 2, d, page)


@pytest.mark.parametrize("layout", ["slots_first", "one_tensor"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_layouts(dev, d, layout):
    run_case(dev, 5, [70, 9, 300], 2, 3, 4, d, 32, layout=layout)


@pytest.mark.parametrize("lens,q_len,g,hkv,d,page", [
    ([9000], 1, 6, 4, 256, 800), ([20000, 3], 3, 6, 2, 128, 16), ([5000] * 3, 5, 6, 1, 64, 48),
    ([4097, 1, 0, 60, 2500, 12000, 7, 640], 1, 8, 8, 128, 16),
    ([100] * 200, 1, 4, 2, 64, 16), ([1] * 700, 1, 2, 1, 128, 16)])
def test_attention_long_and_ragged(dev, lens, q_len, g, hkv, d, page):
    run_case(dev, 3, lens, q_len, g, hkv, d, page)


def test_attention_large_scores(dev):
    """Scores in the hundreds: one key takes all the weight, others underflow; the maximum moves along the keys."""
    run_case(dev, 8, [700, 1500], 2, 6, 2, 128, 16, q_scale=30.0)


@pytest.mark.parametrize("scale", [0.0, -0.07, 1e-30])
def test_attention_scales(dev, scale):
    """Of either sign, and zero: the mean of the values."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(14)
    lens = [300, 65, 2]
    table, pages = table_for(gen, lens, 16)
    cache = random_cache(gen, pages, 16, 2, 128)
    query = torch.randn(9, 10, 128, device=dev, generator=gen).to(BF16)
    out = kv4_attention(query, cache, torch.tensor(lens, dtype=torch.int32, device=dev), table, 3, scale)
    check_attention(out, query, cache, lens, table, 3, scale)


def test_attention_query_rows_are_apart(dev):
    """A row of NaN, of infinities or of very large values leaves the other rows as they are."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(15)
    lens = [400, 90]
    table, pages = table_for(gen, lens, 16)
    cache = random_cache(gen, pages, 16, 2, 256)
    query = torch.randn(4, 12, 256, device=dev, generator=gen).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    clean = kv4_attention(query, cache, seq, table, 2, 0.06)
    query[0, 3], query[1, 7], query[2, 0, 5], query[3, 11] = float("nan"), float("inf"), 3e38, 1e30
    out = kv4_attention(query, cache, seq, table, 2, 0.06)
    other = torch.ones(4, 12, dtype=torch.bool, device=dev)
    other[0, 3] = other[1, 7] = other[2, 0] = other[3, 11] = False
    assert out[0, 3].isnan().all() and out[1, 7].isnan().all()
    # another row may have the references raised at another tile: the weights' roundings (2^-8 of them, on both sides) and the
    # result's may differ, no more
    _, spread, _ = orc.attention(host(query.nan_to_num(0.0, 0.0, 0.0)), [host(t) for t in cache], lens, host(table), 2, 0.06)
    bound = torch.from_numpy(2 * 2.0 ** -8 * spread).to(dev) + 2 * 2.0 ** -8 * clean.double().abs() + 2.0 ** -16
    assert ((out.double() - clean.double()).abs() <= bound)[other].all()


def test_attention_one_key_rows_are_its_values(dev):
    """With one key the weight is exactly 1."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention, kv4_read
    gen = torch.Generator(device=dev).manual_seed(2)
    cache = random_cache(gen, 3, 16, 2, 256)
    query = torch.randn(1, 12, 256, device=dev, generator=gen).to(BF16)
    out = kv4_attention(query, cache, torch.ones(1, dtype=torch.int32, device=dev),
                        torch.tensor([[2]], dtype=torch.int32, device=dev), 1, 0.1)
    _, v = kv4_read(cache, torch.tensor([32], device=dev))
    assert torch.equal(out.view(2, 6, 256), v.view(2, 1, 256).expand(2, 6, 256))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_ignores_what_is_masked(dev, d):
    """NaN in slots behind a request's end, in whole pages that are no one's, and in keys and values that only the later of a
    request's queries see: those become NaN, in the groups that hold one, and no other."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(4)
    lens, q_len, g, hkv, page = [61, 200, 130, 3], 3, 4, 2, 32
    table, pages = table_for(gen, lens, page, spare=3)
    cache = random_cache(gen, pages, page, hkv, d)
    used = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        for p in range(n):
            used[table[b, p // page], p % page] = True
    for t in cache[2:]:
        t.transpose(1, 2)[~used] = float("nan")
    query = torch.randn(len(lens) * q_len, hkv * g, d, device=dev, generator=gen).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = kv4_attention(query, cache, seq, table, q_len, 0.11)
    assert not out.isnan().any()
    check_attention(out, query, cache, lens, table, q_len, 0.11)
    # request 1: the last token's values of head 0; request 2: the second to last one's keys of head 1; request 3: the last
    # one's values, with rows that see nothing else or nothing at all
    def at(b, p):
        return table[b, p // page].item(), p % page
    (p1, o1), (p2, o2), (p3, o3) = at(1, 199), at(2, 128), at(3, 2)
    cache.v_scale[p1, 0, o1, d // 64 - 1] = float("nan")
    cache.k_scale[p2, 1, o2, 0, 1] = float("nan")
    cache.v_scale[p3, :, o3, 0, 0] = float("inf")
    out = kv4_attention(query, cache, seq, table, q_len, 0.11).view(4, q_len, hkv, g, d)
    nan = out.isnan()
    want = torch.zeros_like(nan)
    want[1, 2, 0, :, d - 64:] = True
    want[2, 1:, 1] = True
    assert torch.equal(nan[:3], want[:3])
    assert not nan[3, :2].any() and not nan[3, :, :, :, 64:].any() and not out[3, 2, :, :, :64].isfinite().any()


def test_attention_pages_that_are_none(dev):
    """Keys on pages outside the cache, and behind the table's width, do not take part; a request without any gives zeros."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(9)
    cache = random_cache(gen, 6, 16, 2, 128)
    table = torch.tensor([[0, -1, 5, 1], [6, 2, 2 ** 31 - 1, -2 ** 31], [-1, -1, -1, 99], [3, 4, 0, 1]], dtype=torch.int32,
                         device=dev)
    lens = [64, 60, 40, 1000]
    query = torch.randn(8, 6, 128, device=dev, generator=gen).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = kv4_attention(query, cache, seq, table, 2, 0.09)
    check_attention(out, query, cache, lens, table, 2, 0.09)
    assert not out[4:6].any()
    none = kv4_attention(query, cache, seq, table[:, :0], 2, 0.09)
    assert none.shape == query.shape and not none.any()


def test_attention_lengths_of_any_value(dev):
    """Lengths at the ends of 32 bits: what the table can place takes part, or nothing."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(10)
    lens = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 64, 1 - 2 ** 31, 70]
    table = torch.randperm(30, generator=gen, device=dev).to(torch.int32).view(5, 6)
    query = torch.randn(15, 8, 128, device=dev, generator=gen).to(BF16)
    cache = random_cache(gen, 30, 16, 2, 128)
    out = kv4_attention(query, cache, torch.tensor(lens, dtype=torch.int32, device=dev), table, 3, 0.09)
    check_attention(out, query, cache, lens, table, 3, 0.09)
    assert not out[3:6].any() and not out[9:12].any()


def test_a_cache_of_no_pages(dev):
    """Nothing is written, zeros are read, rows without keys are zeros."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention, kv4_cache, kv4_read, kv4_write
    cache = kv4_cache(0, 16, 2, 128, dev)
    x, slots = torch.ones(3, 2, 128, dtype=BF16, device=dev), torch.tensor([0, -1, 5], device=dev)
    kv4_write(x, x, slots, cache)
    k, v = kv4_read(cache, slots)
    assert k.shape == x.shape and not k.any() and not v.any()
    lens, table = torch.tensor([5, 0, 40], dtype=torch.int32, device=dev), torch.zeros(3, 2, dtype=torch.int32, device=dev)
    out = kv4_attention(x.repeat(1, 3, 1), cache, lens, table, 1, 0.1)
    assert out.shape == (3, 6, 128) and not out.any()


def test_attention_strided_query_and_out(dev):
    """Views of a larger buffer, rows behind the last request left as they were, the version raised."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(12)
    lens, hkv, g, d = [90, 17], 2, 5, 64
    table, pages = table_for(gen, lens, 16)
    cache = random_cache(gen, pages, 16, hkv, d)
    wide = torch.randn(7, hkv * g + 3, d + 8, device=dev, generator=gen).to(BF16)
    query = wide[:, 1:1 + hkv * g, 8:]
    buf = torch.full((7, hkv * g, 2 * d), 7.0, dtype=BF16, device=dev)
    out = buf[:, :, :d]
    version = out._version
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    assert kv4_attention(query, cache, seq, table, 3, 0.2, out=out) is out and out._version > version
    check_attention(out, query[:6], cache, lens, table, 3, 0.2)
    assert (buf[6] == 7).all() and (buf[:, :, d:] == 7).all()
    odd = torch.randn(6, hkv * g, d + 1, device=dev, generator=gen).to(BF16)[:, :, 1:]     # addresses of two bytes
    check_attention(kv4_attention(odd, cache, seq, table, 3, 0.2), odd, cache, lens, table, 3, 0.2)
    turned = torch.randn(d, 6, hkv * g, device=dev, generator=gen).to(BF16).permute(1, 2, 0)
    check_attention(kv4_attention(turned, cache, seq, table, 3, 0.2), turned, cache, lens, table, 3, 0.2)


def test_attention_far_pages(dev):
    """Pages whose bytes lie more than 2^32 behind the cache's first."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_attention
    gen = torch.Generator(device=dev).manual_seed(6)
    pages, page, hkv, d = (1 << 18) + 5, 16, 8, 256
    small = random_cache(gen, 8, page, hkv, d)
    big = KV4Cache(*(torch.empty((pages, *t.shape[1:]), dtype=t.dtype, device=dev) for t in small))
    ids = torch.tensor([pages - 1, 0, pages - 4, 1 << 17, pages - 2, 77, (1 << 18) - 1, 1 << 18], device=dev)
    for b, s in zip(big, small):
        b[ids] = s
    lens = [100, 20]
    far = torch.zeros(2, 7, dtype=torch.int32, device=dev)
    near = torch.zeros_like(far)
    far[0], near[0] = ids[:7], torch.arange(7)
    far[1, :2], near[1, :2] = ids[6:8], torch.tensor([6, 7])
    query = torch.randn(2, 16, d, device=dev, generator=gen).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    a, b = kv4_attention(query, big, seq, far, 1, 0.06), kv4_attention(query, small, seq, near, 1, 0.06)
    assert torch.equal(a, b)
    check_attention(a, query, small, lens, near, 1, 0.06)


def test_attention_same_bits_every_time(dev):
    """Repeated, on another stream, and in a captured graph replayed with other lengths."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention
    gen = torch.Generator(device=dev).manual_seed(7)
    lens = [3000, 100, 0, 777]
    table, pages = table_for(gen, lens, 16)
    cache = random_cache(gen, pages, 16, 2, 128)
    query = torch.randn(8, 12, 128, device=dev, generator=gen).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    first = kv4_attention(query, cache, seq, table, 2, 0.1)
    for _ in range(3):
        assert torch.equal(kv4_attention(query, cache, seq, table, 2, 0.1), first)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = kv4_attention(query, cache, seq, table, 2, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = kv4_attention(query, cache, seq, table, 2, 0.1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(other, first) and torch.equal(caught, first)
    new = [1, 2900, 50, 770]
    table[0, :1], table[1, :7] = table[0, :1].clone(), table[1, :7].clone()
    small = [min(n, m) for n, m in zip(new, lens)]
    seq.copy_(torch.tensor(small, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check_attention(caught, query, cache, small, table, 2, 0.1)


@pytest.mark.parametrize("size", [2.0 ** 113, 2.0 ** 125.9, 2.0 ** -90])
@pytest.mark.parametrize("d,g,hkv", [(64, 1, 1), (128, 4, 2), (256, 6, 2)])
def test_attention_sums_of_large_and_small_values(dev, d, g, hkv, size):
    """A row's result is a mean of its values: their weighted sums stay within fp32 on the way, with scores that rise along
    the keys by nearly the 2^16 up to which a row's reference stays, in one share and over many CTAs.  (The reference lies 16 to
    32 above a row's maximum, so that the distances to it are off by 2^-19 for their rounding, twice in a mean: 2 ln 2 2^-19 of
    A, within the 2^-18 above.)"""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention, kv4_cache, kv4_read, kv4_write
    gen = torch.Generator(device=dev).manual_seed(d)
    lens, q_len, page = [30, 700, 6000], 2, 16
    table, pages = table_for(gen, lens, page)
    cache = kv4_cache(pages, page, hkv, d, dev)
    n = sum(lens)
    slots = torch.cat([table[b, :-(-m // page)].long().repeat_interleave(page)[:m] * page +
                       torch.arange(m, device=dev) % page for b, m in enumerate(lens)])
    k = 0.1 * torch.randn(n, hkv, d, device=dev, generator=gen)
    k += torch.cat([torch.linspace(0, 1, m, device=dev) for m in lens])[:, None, None]
    v = size * (0.5 + 0.5 * torch.rand(n, hkv, d, device=dev, generator=gen))
    kv4_write(k.to(BF16), v.to(BF16), slots, cache)
    query = (1 + 0.1 * torch.randn(len(lens) * q_len, hkv * g, d, device=dev, generator=gen)).to(BF16)
    out = kv4_attention(query, cache, torch.tensor(lens, dtype=torch.int32, device=dev), table, q_len, 10.0 / d)
    assert out.isfinite().all() and out.min() > 0.4 * size and out.max() < 1.1 * size
    check_attention(out, query, cache, lens, table, q_len, 10.0 / d)


@pytest.mark.parametrize("size", [2.0 ** 118, 2.0 ** 122, 2.0 ** 124, 2.0 ** 125.9])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_values_at_the_end_of_the_range(dev, d, size):
    """Groups that the writer keeps as numbers are numbers wherever they lie: in a tile that some rows do not see whole, in
    one that all rows do, in the last token, and hidden from the first rows of a request."""
    from qwen_a100_fastpath_b200.kv4 import kv4_attention, kv4_read, kv4_write
    gen = torch.Generator(device=dev).manual_seed(d)
    lens, q_len, g, hkv, page = [40, 300, 2], 2, 3, 2, 16
    table, pages = table_for(gen, lens, page)
    cache = random_cache(gen, pages, page, hkv, d)
    places = [(0, 7), (0, 39), (1, 20), (1, 290), (2, 1)]
    slots = torch.tensor([table[b, p // page].item() * page + p % page for b, p in places], device=dev)
    k, _ = kv4_read(cache, slots)
    v = (size * (2 * torch.rand(len(places), hkv, d, device=dev, generator=gen) - 1)).to(BF16)
    v[..., 0], v[..., 1] = size, -size
    kv4_write(k, v, slots, cache)
    assert kv4_read(cache, slots)[1].isfinite().all()
    query = torch.randn(len(lens) * q_len, hkv * g, d, device=dev, generator=gen).to(BF16)
    out = kv4_attention(query, cache, torch.tensor(lens, dtype=torch.int32, device=dev), table, q_len, d ** -0.5)
    assert out.isfinite().all()
    check_attention(out, query, cache, lens, table, q_len, d ** -0.5)


# ---- writer and reader --------------------------------------------------------------------------------------------
def tokens(gen, t, hkv, d):
    x = torch.randn(t, hkv, d, device=gen.device, generator=gen) * torch.exp(
        2 * torch.randn(t, hkv, 1, device=gen.device, generator=gen))
    return (x + 3 * torch.randn(t, 1, 1, device=gen.device, generator=gen)).to(BF16)


def check_written(cache, before, k, v, slots):
    """Exactly the slots given hold what the definition says, everything else is untouched."""
    page, n = cache.k.shape[2], cache.k.shape[0] * cache.k.shape[2]
    for x, codes, scale, c0, s0 in ((k, cache.k, cache.k_scale, before.k, before.k_scale),
                                    (v, cache.v, cache.v_scale, before.v, before.v_scale)):
        want_c, want_s = host(c0).copy(), host(s0).copy()
        nib, sc = orc.quantize(host(x))
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < n:
                want_c[slot // page, :, slot % page] = orc.pack(nib[i])
                want_s[slot // page, :, slot % page] = sc[i]
        assert np.array_equal(host(codes), want_c)
        assert np.array_equal(host(scale), want_s, equal_nan=True)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t,hkv,page,layout", [(1, 1, 16, "plain"), (5, 4, 800, "plain"), (333, 3, 7, "slots_first"),
                                               (257, 8, 16, "one_tensor")])
def test_write_and_read(dev, d, t, hkv, page, layout):
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_read, kv4_write
    gen = torch.Generator(device=dev).manual_seed(t)
    pages = -(-t // page) + 2
    cache = random_cache(gen, pages, page, hkv, d, layout)
    before = KV4Cache(*(x.clone() for x in cache))
    k, v = tokens(gen, t, hkv, d), tokens(gen, t, hkv, d)
    slots = torch.randperm(pages * page, generator=gen, device=dev)[:t]
    if t > 4:
        slots[1], slots[3] = -1, pages * page          # padding, and a slot behind the cache
        slots[4] = 2 ** 62
    version = cache.k._version
    kv4_write(k, v, slots, cache)
    assert cache.k._version > version
    check_written(cache, before, k, v, slots)
    rk, rv = kv4_read(cache, slots)
    kept = ((slots >= 0) & (slots < pages * page)).cpu().numpy()
    for x, r in ((k, rk), (v, rv)):
        nib, sc = orc.quantize(host(x))
        want = orc.values(orc.pack(nib), sc)
        want[~kept] = 0
        assert r.shape == x.shape and np.array_equal(host(r), want)
        # and it is near what was written: s / 2 + s / 8 + |lo| / 256, and bf16's rounding of the value
        s = np.repeat(sc[..., 0], 64, -1)
        lo = np.repeat(host(x).reshape(t, hkv, -1, 64).min(-1), 64, -1)
        err = np.abs(want - host(x))[kept]
        assert (err <= (0.625 * s + np.abs(lo) / 256 + np.abs(want) / 256)[kept] * (1 + 1e-6)).all()


@pytest.mark.parametrize("hkv,d", [(1, 64), (4, 64), (3, 128), (3, 256), (8, 256)])
def test_write_and_read_many_tokens(dev, hkv, d):
    """On both sides of the number of tokens from which a CTA takes several times as many, none a multiple of what it takes."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_read, kv4_write
    gen = torch.Generator(device=dev).manual_seed(hkv * d)
    page, per_pass = 16, max(1, 256 // (hkv * d // 4))
    edge = 4 * 4 * 148 * per_pass
    for t in (edge - 1, edge, edge + 2 * per_pass + 1):
        pages = t // page + 2
        cache = random_cache(gen, pages, page, hkv, d)
        before = KV4Cache(*(x.clone() for x in cache))
        k, v = tokens(gen, t, hkv, d), tokens(gen, t, hkv, d)
        slots = torch.randperm(pages * page, generator=gen, device=dev)[:t]
        slots[7], slots[t - 1] = -5, pages * page
        kv4_write(k, v, slots, cache)
        check_written(cache, before, k, v, slots)
        kept = ((slots >= 0) & (slots < pages * page)).cpu().numpy()
        for x, r in zip((k, v), kv4_read(cache, slots)):
            nib, sc = orc.quantize(host(x))
            want = orc.values(orc.pack(nib), sc)
            want[~kept] = 0
            assert np.array_equal(host(r), want)


def test_write_edges(dev):
    """Groups of one value, of zeros, with NaN and infinities, at the ends of the range and among the subnormals."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_cache, kv4_read, kv4_write
    cache = kv4_cache(1, 64, 1, 64, dev)
    before = KV4Cache(*(x.clone() for x in cache))
    rows = torch.zeros(24, 64, dtype=torch.float32, device=dev)
    base = torch.linspace(-1, 1, 64, device=dev)
    rows[1] = 3.0
    rows[2, 7] = float("nan")
    rows[3, 63] = float("inf")
    rows[4, 0] = float("-inf")
    rows[5] = base * 2.0 ** 125.9
    rows[6] = base * 2.0 ** 126
    rows[7] = base * 3.3e38
    rows[8] = base * 2.0 ** -120
    rows[9] = base * 2.0 ** -130
    rows[10, 3] = 2.0 ** -133
    rows[11, 3] = 1e-30
    rows[12] = 100 + 0.5 * (torch.arange(64, device=dev) % 2)
    rows[13] = -1e6 + base
    rows[14] = torch.arange(64, device=dev) % 16
    rows[15] = (torch.arange(64, device=dev) % 31) / 2          # halves: ties
    rows[16] = -((torch.arange(64, device=dev) % 31) / 2)
    rows[17:] = torch.randn(7, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    k = rows.to(BF16)[:, None]
    v = -k.flip(0)
    slots = torch.arange(24, device=dev) + 20
    kv4_write(k, v, slots, cache)
    check_written(cache, before, k, v, slots)
    rk, _ = kv4_read(cache, slots)
    nan = rk.isnan()[:, 0]
    assert nan.any(1).tolist() == [i in (2, 3, 4, 6, 7) for i in range(24)] and nan[[2, 3, 4, 6, 7]].all()
    assert torch.equal(rk[1], k[1]) and not rk[0].any() and torch.equal(rk[14], k[14])


def test_write_strided(dev):
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_write
    gen = torch.Generator(device=dev).manual_seed(3)
    cache = random_cache(gen, 9, 16, 2, 128)
    qkv = tokens(gen, 40, 10, 128)
    for k, v in ((qkv[:, 3:5], qkv[:, 7:9]),                                   # views of the product's rows
                 (qkv[:, 1:2].expand(40, 2, 128), qkv[:, :4:2]),               # one key head for all, every other row
                 (tokens(gen, 40, 2, 129)[..., 1:], tokens(gen, 2, 40, 128).transpose(0, 1))):
        before = KV4Cache(*(x.clone() for x in cache))
        slots = torch.randperm(144, generator=gen, device=dev)[:80][::2]
        kv4_write(k, v, slots, cache)
        check_written(cache, before, k, v, slots)


def at_odd_address(x):
    """The same values, contiguous, two bytes behind a 16-byte boundary."""
    buf = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    buf[1:] = x.reshape(-1)
    return buf[1:].view(x.shape)


@pytest.mark.parametrize("t,hkv,d", [(1, 1, 64), (1, 2, 256), (9, 1, 128), (40, 2, 128)])
def test_contiguous_heads_at_odd_addresses(dev, t, hkv, d):
    """They are copied like other heads that are not aligned: keys, values and the query, each alone and together; a slice of
    a single token and head counts as contiguous whatever its strides."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_attention, kv4_write
    gen = torch.Generator(device=dev).manual_seed(t)
    cache = random_cache(gen, 9, 16, hkv, d)
    k, v = tokens(gen, t, hkv, d), tokens(gen, t, hkv, d)
    for a, b in ((at_odd_address(k), v), (k, at_odd_address(v)), (at_odd_address(k), at_odd_address(v)),
                 (tokens(gen, t, hkv, d + 1)[..., 1:], v)):
        before = KV4Cache(*(x.clone() for x in cache))
        slots = torch.randperm(144, generator=gen, device=dev)[:t]
        kv4_write(a, b, slots, cache)
        check_written(cache, before, a, b, slots)
    lens = [30] * t
    table, pages = table_for(gen, lens, 16)
    cache = random_cache(gen, pages, 16, hkv, d)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    for query in (at_odd_address(tokens(gen, t, hkv, d)), torch.randn(t, hkv, d + 1, device=dev, generator=gen).to(BF16)[..., 1:]):
        got = kv4_attention(query, cache, seq, table, 1, 0.05)
        check_attention(got, query, cache, lens, table, 1, 0.05)
        out = torch.empty(query.shape, dtype=BF16, device=dev)
        assert torch.equal(kv4_attention(query, cache, seq, table, 1, 0.05, out=out), got)


def test_write_far_pages(dev):
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_read, kv4_write
    gen = torch.Generator(device=dev).manual_seed(3)
    pages, page = (1 << 18) + 3, 16
    cache = KV4Cache(*(torch.empty(pages, 8, page, *s, dtype=t, device=dev) for s, t in
                       (((128,), torch.uint8), ((128,), torch.uint8), ((4, 2), BF16), ((4, 2), BF16))))
    k, v = tokens(gen, 20, 8, 256), tokens(gen, 20, 8, 256)
    slots = pages * page - 1 - torch.arange(20, device=dev) * 3
    kv4_write(k, v, slots, cache)
    for x, r in zip((k, v), kv4_read(cache, slots)):
        nib, sc = orc.quantize(host(x))
        assert np.array_equal(host(r), orc.values(orc.pack(nib), sc))


def side_by_side(dev, pages, hkv, page, d, how):
    """Keys and values, and their scales, as views of shared buffers without a common byte."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache
    half, g = d // 2, d // 64
    if how == "slot":
        codes = torch.zeros(pages, hkv, page, 2, half, dtype=torch.uint8, device=dev)
        scale = torch.zeros(pages, hkv, page, 2, g, 2, dtype=BF16, device=dev)
        return KV4Cache(codes[:, :, :, 0], codes[:, :, :, 1], scale[:, :, :, 0], scale[:, :, :, 1])
    if how == "head":
        codes = torch.zeros(pages, hkv, 2, page, half, dtype=torch.uint8, device=dev)
        scale = torch.zeros(pages, hkv, 2, page, g, 2, dtype=BF16, device=dev)
        return KV4Cache(codes[:, :, 0], codes[:, :, 1], scale[:, :, 0], scale[:, :, 1])
    if how == "slots_first":
        codes = torch.zeros(pages, page, hkv, 2, half, dtype=torch.uint8, device=dev).transpose(1, 2)
        scale = torch.zeros(pages, page, 2, hkv, g, 2, dtype=BF16, device=dev).transpose(1, 3)
        return KV4Cache(codes[:, :, :, 0], codes[:, :, :, 1], scale[:, :, 0], scale[:, :, 1])
    # all four in one record for each head and slot
    record = 2 * half + 8 * g + (-8 * g) % 16
    raw = torch.zeros(pages, hkv, page, record, dtype=torch.uint8, device=dev)
    parts = [raw[..., 2 * half + 4 * g * i:2 * half + 4 * g * (i + 1)].view(BF16).unflatten(-1, (g, 2)) for i in range(2)]
    return KV4Cache(raw[..., :half], raw[..., half:2 * half], *parts)


@pytest.mark.parametrize("how", ["slot", "head", "slots_first", "record"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_keys_and_values_side_by_side(dev, d, how):
    """Written (both ways), read and attended like a cache of four buffers."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_attention, kv4_read, kv4_write
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    gen = torch.Generator(device=dev).manual_seed(d)
    pages, hkv, page, g, t = 7, 3, 5, 2, 30
    cache = side_by_side(dev, pages, hkv, page, d, how)
    plain = KV4Cache(*(x.clone(memory_format=torch.contiguous_format) for x in cache))
    k, v = tokens(gen, t, hkv, d), tokens(gen, t, hkv, d)
    slots = torch.randperm(pages * page, generator=gen, device=dev)[:t]
    before = KV4Cache(*(x.clone() for x in cache))
    for c in (cache, plain):
        kv4_write(k, v, slots, c)
    check_written(cache, before, k, v, slots)
    query = tokens(gen, t, hkv * g, d)
    before = KV4Cache(*(x.clone() for x in cache))
    qk_norm_rope(query, v, None, None, None, None, v=k, cache=cache, slots=slots)
    check_written(cache, before, v, k, slots)
    for c in (cache, plain):
        kv4_write(k, v, slots, c)
    table = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)[None]
    lens = torch.tensor([33], dtype=torch.int32, device=dev)
    a, b = (kv4_attention(query, c, lens, table, 1, 0.1) for c in (cache, plain))
    assert torch.equal(a, b)
    for x, y in zip(kv4_read(cache, slots), kv4_read(plain, slots)):
        assert torch.equal(x, y)


# ---- a step as it is used ------------------------------------------------------------------------------------------
def test_step_of_a_layer(dev):
    """Maps from lengths, norms and rotation into the cache, attention: several steps of growing requests, eagerly and as
    one captured graph, against float64 at every stage; and the fused write against the two calls it replaces."""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_attention, kv4_cache, kv4_read, kv4_write
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    from qwen_a100_fastpath_b200.paged import step_maps
    gen = torch.Generator(device=dev).manual_seed(21)
    B, q_len, hkv, g, d, page, rot, pages = 5, 3, 2, 6, 256, 16, 64, 60
    angle = torch.arange(256, device=dev, dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    qw, kw = (0.2 * torch.randn(2, d, device=dev, generator=gen)).to(BF16)
    T = B * q_len + 2                                     # two tokens of padding

    def fresh():
        return dict(past=torch.tensor([0, 1, 13, 60, 14], dtype=torch.int32, device=dev),
                    q=torch.full((B,), q_len, dtype=torch.int32, device=dev),
                    table=torch.full((B, 12), -1, dtype=torch.int32, device=dev),
                    head=torch.zeros(1, dtype=torch.int32, device=dev), cache=kv4_cache(pages, page, hkv, d, dev),
                    qkv=torch.zeros(T, (g + 2) * hkv, d, dtype=BF16, device=dev))

    free = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)

    def step(s, cache):
        m = step_maps(s["q"], s["past"], s["table"], page, T, free_pages=free, free_head=s["head"])
        query, none = qk_norm_rope(s["qkv"][:, :g * hkv], s["qkv"][:, g * hkv:(g + 1) * hkv], qw, kw, m.positions, cos_sin,
                                   weight_offset=1.0, v=s["qkv"][:, (g + 1) * hkv:], cache=cache, slots=m.slots)
        assert none is None
        out = kv4_attention(query, cache, m.seq_lens, s["table"], q_len, d ** -0.5)
        s["head"].copy_(m.free_head)
        s["past"].copy_(m.seq_lens)
        return m, query, out

    eager, caught = fresh(), fresh()
    for s in (eager, caught):   # the pages of what is cached already
        m = step_maps(s["past"], torch.zeros_like(s["past"]), s["table"], page, 0, free_pages=free, free_head=s["head"])
        s["head"].copy_(m.free_head)
    graph = torch.cuda.CUDAGraph()
    start = {k: v.clone() for k, v in caught.items() if torch.is_tensor(v)}
    with torch.cuda.graph(graph):
        result = step(caught, caught["cache"])
    for k, v in start.items():
        caught[k].copy_(v)
    for n in range(6):
        qkv = torch.randn(T, (g + 2) * hkv, d, device=dev, generator=gen).to(BF16)
        eager["qkv"].copy_(qkv)
        caught["qkv"].copy_(qkv)
        past = eager["past"].tolist()
        apart = KV4Cache(*(x.clone() for x in eager["cache"]))
        m, query, out = step(eager, eager["cache"])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*m, query, out, *eager["cache"]), (*result[0], *result[1:], *caught["cache"])):
            assert torch.equal(a, b)
        assert m.seq_lens.tolist() == [p + q_len for p in past]
        assert m.positions.tolist() == [p + i for p in past for i in range(q_len)] + [0, 0]
        # the two calls that the fused one stands for
        q2, k2 = qk_norm_rope(qkv[:, :g * hkv], qkv[:, g * hkv:(g + 1) * hkv], qw, kw, m.positions, cos_sin,
                              weight_offset=1.0)
        kv4_write(k2, qkv[:, (g + 1) * hkv:], m.slots, apart)
        assert torch.equal(q2, query) and all(torch.equal(a, b) for a, b in zip(apart, eager["cache"]))
        nib, sc = orc.quantize(host(k2[:B * q_len]))
        rk, _ = kv4_read(eager["cache"], m.slots)
        assert np.array_equal(host(rk)[:B * q_len], orc.values(orc.pack(nib), sc)) and not rk[B * q_len:].any()
        check_attention(out, query[:B * q_len], eager["cache"], m.seq_lens.tolist(), eager["table"], q_len, d ** -0.5)
    used = eager["table"][eager["table"] >= 0]
    assert used.numel() == used.unique().numel() == int(eager["head"])
