"""The 4-bit cache, the head norms with rotation and the step maps on the CPU: the oracle's own arithmetic, the C ABI's
refusals before any CUDA call, the operators' refusals, and their shapes under tracing."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as orc
from qwen_a100_fastpath_b200 import _lib, kv4, norms, paged

FAKE = 1 << 20
LIB = _lib.LIB
BF16, I32, I64 = torch.bfloat16, torch.int32, torch.int64


# ---- the oracle ------------------------------------------------------------------------------------------------------
def test_round_bf16_is_torchs():
    x = np.random.RandomState(0).standard_normal(20000).astype(np.float32)
    x = np.concatenate([x, x * np.float32(1e-39), x * np.float32(2.0 ** 126), np.float32([0, 1.00390625, 1.01171875, np.inf])])
    t = torch.from_numpy(x).to(BF16).double().numpy()
    assert np.array_equal(orc.round_bf16(x.astype(np.float64)), t)
    assert np.isnan(orc.round_bf16(np.array([np.nan]))).all()


def test_quantizer_of_a_line():
    x = np.arange(64, dtype=np.float64) % 16 - 4
    n, sc = orc.quantize(x)
    assert sc.tolist() == [[1.0, -20.0]] and n.tolist() == [i % 16 for i in range(64)]
    assert np.array_equal(orc.values(orc.pack(n), sc), x)
    assert orc.pack(np.array([1, 2, 15, 0], np.uint8)).tolist() == [0x21, 0x0F]


def test_attention_of_equal_keys_is_the_mean():
    codes = np.zeros((1, 1, 4, 32), np.uint8)
    scale = np.zeros((1, 1, 4, 1, 2))
    vs = scale.copy()
    vs[0, 0, :, 0, 1] = [1, 2, 3, 10]
    out, spread, _ = orc.attention(np.ones((2, 1, 64)), (codes, codes, scale, vs), [3], np.zeros((1, 1), int), 2, 1.0)
    assert np.allclose(out[0], 1.5) and np.allclose(out[1], 2.0) and np.allclose(spread, out)


# ---- the C ABI -------------------------------------------------------------------------------------------------------
def cache_struct(**kw):
    a = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, page_stride=8192, head_stride=2048, slot_stride=128,
             scale_page_stride=512, scale_head_stride=128, scale_slot_stride=8, num_pages=9, page_size=16, num_heads=4,
             head_size=256)
    a.update(kw)
    return ctypes.pointer(_lib.KV4CacheStruct(*a.values()))


def io(fn=LIB.qf_kv4_write, cache=None, **kw):
    a = dict(k=FAKE, sk_t=1024, sk_h=256, v=FAKE, sv_t=1024, sv_h=256, slots=FAKE, tokens=3, cache=cache or cache_struct(),
             flags=0, stream=None)
    a.update(kw)
    return fn(*a.values())


BAD_CACHES = [(dict(num_pages=-1), -2), (dict(page_size=0), -2), (dict(num_heads=0), -2), (dict(head_size=96), -2),
              (dict(k=None), -1), (dict(v_scale=None), -1), (dict(slot_stride=-128), -3), (dict(page_stride=8200), -4),
              (dict(scale_slot_stride=4), -4), (dict(page_stride=1 << 33), -3), (dict(slot_stride=1 << 32), -3),
              (dict(scale_page_stride=1 << 32), -3), (dict(v=FAKE + 8), -4), (dict(k_scale=FAKE + 8), -4)]


@pytest.mark.parametrize("fn", ["write", "read"])
@pytest.mark.parametrize("kw,code", [(dict(tokens=-1), -2), (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1),
                                     (dict(sk_t=-8), -3), (dict(sv_h=4), -4), (dict(k=FAKE + 2), -4), (dict(slots=FAKE + 4), -4),
                                     (dict(tokens=1 << 24), -2)])
def test_io_argument_validation(fn, kw, code):
    f = LIB.qf_kv4_write if fn == "write" else LIB.qf_kv4_read
    assert io(f, **kw) == code and len(LIB.qf_last_error_detail()) > 0
    assert io(f, tokens=0, k=None) == 0


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_cache_validation(kw, code):
    bad = cache_struct(**kw)
    assert io(cache=bad) == code and attn(cache=bad) == code
    assert rope(k_out=None, v=FAKE, slots=FAKE, cache=bad) == code


def attn(**kw):
    a = dict(q=FAKE, sq_t=6144, sq_h=256, cache=cache_struct(), table=FAKE, s_bt=10, max_pages=10, lens=FAKE, out=FAKE,
             so_t=6144, so_h=256, reqs=2, q_len=3, heads=24, scale=0.1, ws=FAKE, ws_bytes=1 << 40, flags=0, stream=None)
    a.update(kw)
    return LIB.qf_kv4_attn(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(reqs=-1), -2), (dict(q_len=0), -2), (dict(heads=25), -2), (dict(q_len=11), -2), (dict(max_pages=-1), -2),
    (dict(heads=65536 * 4), -2), (dict(reqs=1 << 30), -2), (dict(max_pages=1 << 30), -2), (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1),
    (dict(q=None), -1), (dict(out=None), -1), (dict(lens=None), -1), (dict(table=None), -1), (dict(s_bt=-1), -3),
    (dict(sq_t=-8), -3), (dict(sq_h=100), -4), (dict(out=FAKE + 8), -4), (dict(lens=FAKE + 2), -4), (dict(ws=FAKE + 8), -4),
    (dict(ws=None), -6), (dict(ws_bytes=0), -6)])
def test_attention_argument_validation(kw, code):
    assert attn(**kw) == code and len(LIB.qf_last_error_detail()) > 0
    assert attn(reqs=0, q=None) == 0 and attn(heads=0) == 0


def rope(**kw):
    a = dict(q=FAKE, sq_t=8192, sq_h=256, k=FAKE, sk_t=8192, sk_h=256, qw=FAKE, kw=FAKE, offset=0.0, eps=1e-6, pos=FAKE,
             cs=FAKE, s_cs=64, cs_type=1, max_pos=100, rot=64, inter=0, q_out=FAKE, so_t=6144, so_h=256, k_out=FAKE, sp_t=1024,
             sp_h=256, v=None, sv_t=0, sv_h=0, slots=None, cache=None, tokens=3, heads=24, kv_heads=4, d=256, flags=0,
             stream=None)
    a.update(kw)
    return LIB.qf_qk_norm_rope(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), -2), (dict(heads=-1), -2), (dict(kv_heads=-1), -2), (dict(d=0), -2), (dict(d=513), -2),
    (dict(rot=63), -2), (dict(rot=258), -2), (dict(rot=-2), -2), (dict(max_pos=-1), -2), (dict(tokens=1 << 30), -2),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(cs_type=2), -8), (dict(s_cs=-1), -3), (dict(so_h=-256), -3),
    (dict(q=None), -1), (dict(k=None), -1), (dict(q_out=None), -1), (dict(k_out=None), -1), (dict(pos=None), -1),
    (dict(cs=None), -1), (dict(q=FAKE + 1), -4), (dict(cs=FAKE + 2), -4), (dict(pos=FAKE + 4), -4),
    (dict(cache=cache_struct()), -1), (dict(cache=cache_struct(), k_out=None, v=FAKE), -1),
    (dict(cache=cache_struct(), v=FAKE, slots=FAKE), -1), (dict(cache=cache_struct(num_heads=2), k_out=None), -2),
    (dict(cache=cache_struct(head_size=128), k_out=None), -2)])
def test_rope_argument_validation(kw, code):
    assert rope(**kw) == code and len(LIB.qf_last_error_detail()) > 0
    assert rope(tokens=0, q=None) == 0 and rope(heads=0, kv_heads=0) == 0


def maps(**kw):
    a = dict(q=FAKE, past=FAKE, reqs=3, table=FAKE, s_bt=8, width=8, page=16, free=FAKE, n_free=5, head=FAKE, start=FAKE,
             seq=FAKE, pos=FAKE, slots=FAKE, tokens=7, head_out=FAKE, flags=0, stream=None)
    a.update(kw)
    return LIB.qf_step_maps(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(reqs=-1), -2), (dict(reqs=16385), -2), (dict(width=-1), -2), (dict(n_free=-1), -2), (dict(tokens=-1), -2),
    (dict(page=0), -2), (dict(s_bt=7), -3), (dict(q=None), -1), (dict(past=None), -1), (dict(table=None), -1),
    (dict(start=None), -1), (dict(seq=None), -1), (dict(pos=None), -1), (dict(slots=None), -1), (dict(free=None), -1),
    (dict(head=None), -1), (dict(head_out=None), -1), (dict(head=None, head_out=None), -1), (dict(q=FAKE + 2), -4),
    (dict(pos=FAKE + 4), -4)])
def test_maps_argument_validation(kw, code):
    assert maps(**kw) == code and len(LIB.qf_last_error_detail()) > 0


# ---- the operators' refusals ------------------------------------------------------------------------------------------
def cpu_cache(pages=4, page=16, heads=2, d=128, device="cpu"):
    return kv4.kv4_cache(pages, page, heads, d, device=device)


def test_cpu_tensors_are_refused():
    c = cpu_cache()
    k = torch.zeros(3, 2, 128, dtype=BF16)
    slots = torch.zeros(3, dtype=I64)
    lens, table = torch.ones(3, dtype=I32), torch.zeros(3, 1, dtype=I32)
    for call in (lambda: kv4.kv4_write(k, k, slots, c), lambda: kv4.kv4_read(c, slots),
                 lambda: kv4.kv4_attention(k, c, lens, table, 1, 0.1),
                 lambda: kv4.kv4_attention(k, c, lens, table, 1, 0.1, out=torch.empty_like(k)),
                 lambda: norms.qk_norm_rope(k, k, None, None, None, None),
                 lambda: norms.qk_norm_rope(k, k, None, None, None, None, v=k, cache=c, slots=slots),
                 lambda: paged.step_maps(lens, lens, table, 16, 3),
                 lambda: paged.step_maps(lens, lens, table, 16, 3, free_pages=lens, free_head=lens[:1])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def with_(base, **kw):
    d = dict(base)
    d.update(kw)
    return d


META = "meta"


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype, device=META)


WRITE = dict(k=z(3, 2, 128), v=z(3, 2, 128), slots=z(3, dtype=I64), cache=cpu_cache(device=META))
ATTN = dict(query=z(6, 8, 128), cache=cpu_cache(device=META), seq_lens=z(3, dtype=I32), block_table=z(3, 4, dtype=I32),
            q_len=2, scale=0.1)
ROPE = dict(q=z(5, 8, 128), k=z(5, 2, 128), q_weight=z(128), k_weight=z(128), positions=z(5, dtype=I64),
            cos_sin=z(50, 64, dtype=torch.float32))
INTO = with_(ROPE, v=z(5, 2, 128), slots=z(5, dtype=I64), cache=cpu_cache(device=META))
MAPS = dict(query_lens=z(3, dtype=I32), past_lens=z(3, dtype=I32), block_table=z(3, 4, dtype=I32), page_size=16,
            num_tokens=9)
GROW = with_(MAPS, free_pages=z(7, dtype=I32), free_head=z(1, dtype=I32))


def other(i, t):
    c = list(cpu_cache(device=META))
    c[i] = t
    return kv4.KV4Cache(*c)


@pytest.mark.parametrize("call,base,change", [
    *[(kv4.kv4_write, WRITE, c) for c in (
        dict(k=z(3, 2, 128, dtype=torch.float16)), dict(k=z(3, 256)), dict(k=z(4, 2, 128)), dict(v=z(3, 1, 128)),
        dict(v=z(3, 2, 64)), dict(slots=z(3, dtype=I32)), dict(slots=z(2, dtype=I64)), dict(slots=z(3, 1, dtype=I64)),
        dict(cache=other(0, z(4, 2, 16, 64))), dict(cache=other(0, z(4, 2, 16, 48, dtype=torch.uint8))),
        dict(cache=other(1, z(5, 2, 16, 64, dtype=torch.uint8))), dict(cache=other(2, z(4, 2, 16, 4))),
        dict(cache=other(2, z(4, 2, 16, 1, 2))), dict(cache=other(3, z(4, 2, 16, 2, 3))),
        dict(cache=other(3, z(4, 2, 16, 2, 2, dtype=torch.float16))))],
    *[(kv4.kv4_attention, ATTN, c) for c in (
        dict(query=z(6, 8, 64)), dict(query=z(6, 7, 128)), dict(query=z(5, 8, 128)), dict(query=z(6, 8, 128, dtype=torch.float16)),
        dict(seq_lens=z(3, dtype=I64)), dict(seq_lens=z(4, dtype=I32)), dict(block_table=z(3, 4, dtype=I64)),
        dict(block_table=z(2, 4, dtype=I32)), dict(block_table=z(3, dtype=I32)), dict(q_len=0), dict(q_len=17),
        dict(q_len=2 ** 40), dict(scale=float("inf")), dict(out=z(6, 8, 64)), dict(out=z(6, 8, 128, dtype=torch.float32)))],
    *[(norms.qk_norm_rope, ROPE, c) for c in (
        dict(q=z(5, 8, 128, dtype=torch.float32)), dict(q=z(6, 8, 128)), dict(k=z(5, 2, 64)), dict(k=z(5, 256)),
        dict(q_weight=z(64)), dict(k_weight=z(128, dtype=torch.float32)), dict(positions=z(4, dtype=I64)),
        dict(positions=z(5, dtype=I32)), dict(positions=None), dict(cos_sin=z(50, 63, dtype=torch.float32)),
        dict(cos_sin=z(50, 130, dtype=torch.float32)), dict(cos_sin=z(50, 64, dtype=torch.float16)),
        dict(cos_sin=z(64, dtype=torch.float32)), dict(eps=-1.0), dict(eps=float("nan")), dict(v=z(5, 2, 128)))],
    *[(norms.qk_norm_rope, INTO, c) for c in (
        dict(v=z(4, 2, 128)), dict(slots=z(5, dtype=I32)), dict(k=z(5, 4, 128)), dict(slots=None),
        dict(cache=other(0, z(4, 2, 16, 32, dtype=torch.uint8))))],
    *[(paged.step_maps, MAPS, c) for c in (
        dict(query_lens=z(3, dtype=I64)), dict(past_lens=z(2, dtype=I32)), dict(block_table=z(2, 4, dtype=I32)),
        dict(block_table=z(3, 4, dtype=I64)), dict(page_size=0), dict(page_size=2 ** 31), dict(num_tokens=-1),
        dict(num_tokens=2 ** 31), dict(free_pages=z(7, dtype=I32)))],
    *[(paged.step_maps, GROW, c) for c in (
        dict(free_pages=z(7, dtype=I64)), dict(free_head=z(2, dtype=I32)), dict(free_head=z(1, dtype=I64)))]])
def test_shapes_and_types_are_refused(call, base, change):
    call(**base)
    with pytest.raises(ValueError):
        call(**with_(base, **change))


def test_results_of_traced_calls():
    assert kv4.kv4_write(**WRITE) is None
    k, v = kv4.kv4_read(WRITE["cache"], WRITE["slots"])
    assert k.shape == v.shape == (3, 2, 128) and k.dtype == BF16
    assert kv4.kv4_attention(**with_(ATTN, query=z(8, 8, 128))).shape == (6, 8, 128)
    out = z(6, 8, 128)
    assert kv4.kv4_attention(**ATTN, out=out) is out
    q, k = norms.qk_norm_rope(**ROPE)
    assert q.shape == (5, 8, 128) and k.shape == (5, 2, 128)
    q, none = norms.qk_norm_rope(**INTO)
    assert q.shape == (5, 8, 128) and none is None
    m = paged.step_maps(**GROW)
    assert [(t.shape[0], t.dtype) for t in m] == [(4, I32), (3, I32), (9, I64), (9, I64), (1, I32)]
    assert paged.step_maps(**MAPS).free_head is None


def test_the_token_count_stays_symbolic():
    from torch.fx.experimental.proxy_tensor import make_fx
    c, cs, table = cpu_cache(), torch.zeros(50, 64), torch.zeros(9, 4, dtype=I32)

    def step(qkv, lens):
        pos = torch.zeros(qkv.shape[0], dtype=I64)
        m = paged.step_maps(lens, lens, table[:lens.shape[0]], 16, 9)
        q, _ = norms.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], None, None, pos, cs, v=qkv[:, 6:], cache=c, slots=pos)
        kv4.kv4_write(qkv[:, 4:6], qkv[:, 6:], pos, c)
        k, _ = kv4.kv4_read(c, pos)
        return kv4.kv4_attention(q, c, m.seq_lens, table, 1, 0.1), k

    gm = make_fx(step, tracing_mode="symbolic", _allow_non_fake_inputs=True)(torch.zeros(7, 8, 128, dtype=BF16),
                                                                             torch.zeros(5, dtype=I32))
    out = next(n for n in gm.graph.nodes if n.op == "output").args[0]
    for n in out:
        size = n.meta["val"].shape[0]
        assert isinstance(size, torch.SymInt) and not size.node.expr.is_number, n


def test_gradients_and_tangents_are_refused():
    lead = dict(WRITE, cache=cpu_cache(device=META))
    with pytest.raises(ValueError, match="gradient"):
        kv4.kv4_write(**with_(lead, k=z(3, 2, 128).requires_grad_()))
    with pytest.raises(ValueError, match="gradient"):
        kv4.kv4_attention(**with_(ATTN, query=z(6, 8, 128).requires_grad_()))
    with pytest.raises(ValueError, match="gradient"):
        norms.qk_norm_rope(**with_(ROPE, k_weight=z(128).requires_grad_()))
    with torch.no_grad():
        norms.qk_norm_rope(**with_(ROPE, k_weight=z(128).requires_grad_()))
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda q: norms.qk_norm_rope(**with_(ROPE, q=q))[0], (z(5, 8, 128),), (z(5, 8, 128),))


def test_new_caches():
    c = cpu_cache(3, 7, 5, 256)
    assert c.k.shape == c.v.shape == (3, 5, 7, 128) and c.k_scale.shape == c.v_scale.shape == (3, 5, 7, 4, 2)
    for bad in ((3, 7, 5, 96), (-1, 7, 5, 64), (3, 0, 5, 64), (3, 7, 0, 64)):
        with pytest.raises(ValueError):
            kv4.kv4_cache(*bad, device="cpu")
