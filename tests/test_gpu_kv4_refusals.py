"""Calls of the 4-bit cache's operators that name memory they must not share or cannot take: refused before anything is
written."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_overlap import refused

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_cache_memory(dev):
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_cache, kv4_read, kv4_write
    from qwen_a100_fastpath_b200.norms import qk_norm_rope
    c = kv4_cache(4, 16, 2, 128, dev)
    k = torch.ones(5, 2, 128, dtype=BF16, device=dev)
    slots = torch.arange(5, device=dev)

    def both(cache, k=k, v=k, slots=slots):
        return (lambda: kv4_write(k, v, slots, cache),
                lambda: qk_norm_rope(k, k, None, None, None, None, v=v, cache=cache, slots=slots))

    shared = torch.zeros(4 * 2 * 16 * 64 + 16, dtype=torch.uint8, device=dev)
    shape = c.k.shape
    for bad in (KV4Cache(c.k, c.k, c.k_scale, c.v_scale), KV4Cache(c.k, c.v, c.k_scale, c.k_scale),
                KV4Cache(shared[:-16].view(shape), shared[16:].view(shape), c.k_scale, c.v_scale),
                KV4Cache(c.k[:1].expand(shape), c.v[:1].expand(shape), c.k_scale, c.v_scale),     # a page written for all
                KV4Cache(c.k, c.v, c.k_scale[:, :, :1].expand_as(c.k_scale), c.v_scale[:, :, :1].expand_as(c.v_scale))):
        for call in both(bad):
            refused(call)
    raw = c.k.view(-1).view(BF16)
    for call in both(c, v=raw[:5 * 256].view(5, 2, 128)):
        refused(call)
    for call in both(c, slots=c.v.view(-1)[80:160].view(torch.int64)[:5]):
        refused(call)
    refused(lambda: qk_norm_rope(k, k, raw[:128], None, None, None, v=k, cache=c, slots=slots))
    assert not c.k.any() and not c.v.any() and not c.k_scale.any()
    # what cannot be addressed: strides that differ, rows that are not adjacent or not aligned
    wide = torch.zeros(4, 2, 16, 72, dtype=torch.uint8, device=dev)
    for bad in (KV4Cache(wide[..., :64], c.v, c.k_scale, c.v_scale), KV4Cache(wide[..., :64], wide[..., 8:], c.k_scale, c.v_scale),
                KV4Cache(wide[..., 8:], wide.clone()[..., 8:], c.k_scale, c.v_scale),
                KV4Cache(c.k.transpose(2, 3).contiguous().transpose(2, 3), c.v.transpose(2, 3).contiguous().transpose(2, 3),
                         c.k_scale, c.v_scale),
                KV4Cache(c.k.cpu(), c.v, c.k_scale, c.v_scale)):
        for call in (*both(bad), lambda: kv4_read(bad, slots)):
            with pytest.raises(ValueError):
                call()
    kv4_read(KV4Cache(c.k, c.k, c.k_scale, c.k_scale), slots)             # reading one side twice is fine


@pytest.mark.parametrize("shift", [16, 48, 64, 80, 112])
def test_caches_whose_rows_meet(dev, shift):
    """Values that begin inside the keys' rows, or whose rows reach into the next keys: side by side only at the row's end.
    (Ones are a step of 0, an offset of 1 and nibbles of 0: what a call wrote is seen in the offsets.)"""
    from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_cache, kv4_write
    c = kv4_cache(3, 4, 2, 128, dev)
    k = torch.ones(5, 2, 128, dtype=BF16, device=dev)
    slots = torch.arange(5, device=dev)
    for lead in ((3, 2, 4), (3, 4, 2)):
        raw = torch.zeros(3 * 2 * 4 * 128 + 128, dtype=torch.uint8, device=dev)
        rows = [raw[at:at + 3072].view(*lead, 128)[..., :64] for at in (0, shift)]
        if lead[1] == 4:
            rows = [r.transpose(1, 2) for r in rows]
        cache = KV4Cache(rows[0], rows[1], c.k_scale, c.v_scale)
        if shift == 64:
            kv4_write(k, k, slots, cache)
            assert (c.k_scale[0, :, :, :, 1] == 1).all() and torch.equal(c.v_scale, c.k_scale)
            c.k_scale.zero_(), c.v_scale.zero_()
        else:
            refused(lambda: kv4_write(k, k, slots, cache))
            assert not c.k_scale.any() and not c.v_scale.any()
    # the same on the level of heads: the values' page of heads begins one head late
    raw = torch.zeros(3 * 2 * 2 * 4 * 64 + 1024, dtype=torch.uint8, device=dev)
    rows = [raw[at:at + 3072].view(3, 2, 2, 4, 64)[:, :, 0] for at in (0, 512, 256)]
    refused(lambda: kv4_write(k, k, slots, KV4Cache(rows[0], rows[1], c.k_scale, c.v_scale)))
    assert not c.k_scale.any() and not c.v_scale.any()
    kv4_write(k, k, slots, KV4Cache(rows[0], rows[2], c.k_scale, c.v_scale))
    assert (c.k_scale[0, :, :, :, 1] == 1).all()


def test_attention_memory(dev):
    from qwen_a100_fastpath_b200.kv4 import kv4_attention, kv4_cache
    c = kv4_cache(4, 16, 2, 128, dev)
    buf = torch.zeros(9, 8, 128, dtype=BF16, device=dev)
    lens, table = torch.ones(4, dtype=torch.int32, device=dev), torch.zeros(4, 2, dtype=torch.int32, device=dev)
    q = torch.ones(4, 8, 128, dtype=BF16, device=dev)

    def call(query, out, **kw):
        return kv4_attention(query, c, kw.get("lens", lens), kw.get("table", table), 1, 0.1, out=out)

    refused(lambda: call(buf[:4], buf[3:7]))
    refused(lambda: call(buf[:4], buf[:4]))
    refused(lambda: call(q, c.v.view(-1).view(BF16)[:4096].view(4, 8, 128)))
    refused(lambda: call(q, buf[:4], lens=buf.view(-1)[:8].view(torch.int32)))
    refused(lambda: call(q, buf[:4], table=buf.view(-1)[16:32].view(torch.int32).view(4, 2)))
    for out in (buf[:1].expand(4, 8, 128), torch.zeros(4, 8, 256, dtype=BF16, device=dev)[..., ::2],
                torch.zeros(4, 8, 132, dtype=BF16, device=dev)[..., :128], torch.zeros(4 * 1024 + 1, dtype=BF16,
                                                                                      device=dev)[1:].view(4, 8, 128)):
        with pytest.raises(ValueError):
            call(q, out)
    assert not buf.any()
    call(buf[:4], buf[4:8])


def test_table_memory(dev):
    from qwen_a100_fastpath_b200.paged import step_maps
    buf = torch.arange(64, dtype=torch.int32, device=dev)
    q, past, free, head = (torch.ones(n, dtype=torch.int32, device=dev) for n in (3, 3, 9, 1))

    def call(table, q=q, past=past, free=free, head=head):
        return lambda: step_maps(q, past, table, 16, 5, free_pages=free, free_head=head)

    t = buf[:24].view(3, 8)
    refused(call(t, q=buf[5:8]))
    refused(call(t, past=buf[23:26]))
    refused(call(t, free=buf[20:30]))
    refused(call(t, head=buf[23:24]))
    for bad in (buf[:8].expand(3, 8), buf[:24].view(8, 3).t(), buf[:12].as_strided((3, 8), (2, 1))):
        with pytest.raises(ValueError):
            call(bad)()
    assert torch.equal(buf.cpu(), torch.arange(64, dtype=torch.int32))
    call(t, q=buf[24:27], free=buf[27:40])()
