"""What lies between the qkv product and the attention of a serving step on a paged cache held in 4 bits, as measured:
the maps of a step built on the GPU from the requests' lengths (positions, slots, pages taken from a free list), the norms
of queries and keys for each head with the position rotation (alone, or writing the cache in the same pass), the cache's
writer with its reader, and the attention that reads the cache.

``run`` computes them in elementary torch operations where ``own`` is false, and through this package's public entry
points where it is true.  Sizes are this repository's attention layer (24 query and 4 key heads of 256, pages of 800
slots, verification batches of a few tokens at up to 100K) and, in ``draw``, everything around it.

The cache's format: ``k`` and ``v`` uint8 ``[pages, heads, slots, D / 2]`` (the even dimension in the low nibble), each
with bf16 ``[pages, heads, slots, D / 64, 2]``, the step ``s`` and offset ``c`` of 64 consecutive dimensions; a nibble
``n`` stands for ``bf16((n + 16) s + c)``.
"""
import math

import torch

own = False

GROUP = 64
EPS = 1e-6


def listed():
    return [
        # the verification step of one request (a token and four drafts), which grows into a new page now and then
        dict(name="maps_verify", kind="maps", b=1, q="five", tokens=5, page=800, past=40000),
        # a batch of decoding requests with some prompt chunks among them, padded to a captured size
        dict(name="maps_mixed", kind="maps", b=256, q="mixed", tokens=8192, page=16, past=8192),
        # prompts arriving together: many tokens, most pages new
        dict(name="maps_prompts", kind="maps", b=1024, q="long", tokens=131072, page=64, past=512),
        # queries and keys of a verification batch, keys and values straight into the cache: a layer's latency counts
        dict(name="rope_verify", kind="rope", t=5, h=24, hkv=4, d=256, rot=64, inter=False, norm=True, offset=1.0,
             table="f32", cache=True, page=800, fused_qkv=True),
        # other heads: full rotation of interleaved pairs, a bf16 table, no size a multiple of a tile
        dict(name="rope_ragged", kind="rope", t=333, h=40, hkv=8, d=128, rot=128, inter=True, norm=True, offset=0.0,
             table="bf16", cache=False, page=16, fused_qkv=True),
        # a whole prompt, queries and keys returned
        dict(name="rope_prompt", kind="rope", t=8192, h=24, hkv=4, d=256, rot=64, inter=False, norm=True, offset=1.0,
             table="f32", cache=False, page=800, fused_qkv=True),
        # keys and values of a decoding batch into the cache and back
        dict(name="cache_batch", kind="cache", t=64, hkv=4, d=256, page=800),
        # the same for a prompt chunk on small pages
        dict(name="cache_prompt", kind="cache", t=8192, hkv=8, d=128, page=16),
        # one token of a short chat
        dict(name="attn_token", kind="attn", b=1, q=1, h=24, hkv=4, d=256, page=800, longest=700, ragged=False),
        # a verification step of one request at 38K context
        dict(name="attn_verify", kind="attn", b=1, q=3, h=24, hkv=4, d=256, page=800, longest=38400, ragged=False),
        # a decoding batch of very different lengths on small pages, other heads
        dict(name="attn_batch", kind="attn", b=64, q=1, h=64, hkv=8, d=128, page=16, longest=8192, ragged=True),
        # two verification steps at 100K context
        dict(name="attn_long", kind="attn", b=2, q=5, h=24, hkv=4, d=256, page=800, longest=100000, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _page(rng):
    return rng.choice((16, 32, 64, 128, 800, rng.randint(1, 300)))


def draw(rng):
    kind = rng.choice(("maps", "rope", "cache", "attn", "attn"))
    if kind == "maps":
        b = _log_int(rng, 1, 1024)
        q = rng.choice(("one", "five", "mixed", "long"))
        need = {"one": b, "five": 5 * b}.get(q, b + _log_int(rng, 1, 131072 - 1024))
        # a token map is often padded to a captured size
        tokens = need if rng.random() < 0.5 else min(131072, need + _log_int(rng, 1, 4096))
        return dict(kind="maps", b=b, q=q, tokens=tokens, page=max(_page(rng), 8 if b > 64 else 1),
                    past=_log_int(rng, 1, 40000 if b <= 64 else 8192))
    if kind == "attn":
        d = rng.choice((64, 128, 256))
        hkv = rng.choice((1, 2, 4, 8, rng.randint(1, 12)))
        q = rng.choice((1, 1, rng.randint(1, 8)))
        g = rng.randint(1, 64 // q if q > 3 else 16)
        b = _log_int(rng, 1, 96)
        ragged = rng.random() < 0.5
        longest = _log_int(rng, q, 100000)
        # no more of the cache, and no more rows for each key, than the largest listed case
        while b * longest * hkv * d * max(1.0, q * g / 30) > 2 * 100000 * 4 * 256:
            if longest > 64 and (b == 1 or rng.random() < 0.5):
                longest = max(q, longest // 2)
            elif b > 1:
                b //= 2
            else:
                break
        return dict(kind="attn", b=b, q=q, h=hkv * g, hkv=hkv, d=d, page=_page(rng), longest=longest, ragged=ragged)
    if kind == "cache":
        t, hkv, d = _log_int(rng, 1, 16384), rng.randint(1, 16), rng.choice((64, 128, 256))
        while t * hkv * d > 8192 * 8 * 128:
            t //= 2
        return dict(kind="cache", t=t, hkv=hkv, d=d, page=_page(rng))
    cache = rng.random() < 0.4
    d = rng.choice((64, 128, 256) if cache else (64, 80, 96, 128, 192, 256))
    t, hkv = _log_int(rng, 1, 16384), rng.choice((1, 2, 4, 8))
    h = hkv * rng.randint(1, 8)
    while t * (h + hkv) * d > 8192 * 28 * 256:
        t //= 2
    rot = d if rng.random() < 0.5 else rng.choice((16, 20, 32, 48, 64))
    return dict(kind="rope", t=t, h=h, hkv=hkv, d=d, rot=rot, inter=rng.random() < 0.3, norm=rng.random() < 0.8,
                offset=rng.choice((0.0, 1.0)), table=rng.choice(("f32", "f32", "bf16")), cache=cache, page=_page(rng),
                fused_qkv=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _up(a, b):
    return -(-a // b)


def _heads(gen, t, heads, d):
    """Rows of a qkv product: normal values, channels of different sizes in each head, some of them much larger."""
    x = torch.randn((t, heads, d), generator=gen, device=gen.device)
    x *= torch.exp(0.5 * torch.randn((heads, d), generator=gen, device=gen.device))
    loud = torch.rand((heads, d), generator=gen, device=gen.device) < 0.01
    x *= torch.where(loud, 6.0, 1.0)
    x += 0.3 * torch.randn((heads, d), generator=gen, device=gen.device)
    return x.to(torch.bfloat16)


def _empty_cache(pages, page, hkv, d):
    def half():
        return (torch.zeros((pages, hkv, page, d // 2), dtype=torch.uint8, device=_dev()),
                torch.zeros((pages, hkv, page, d // GROUP, 2), dtype=torch.bfloat16, device=_dev()))
    (k, ks), (v, vs) = half(), half()
    return k, v, ks, vs


def _slots(gen, t, page, pages):
    """Slots of t tokens as requests leave them: runs inside pages in any order, some tokens of padding."""
    order = torch.randperm(pages, generator=gen, device=gen.device)
    i = torch.arange(t, device=gen.device)
    slots = order[i // page] * page + i % page
    if t >= 16:
        slots[-(t // 16):] = -1
    return slots


def _query_lens(case, gen):
    b, tokens = case["b"], case["tokens"]
    if case["q"] in ("one", "five"):
        return torch.full((b,), 1 if case["q"] == "one" else 5, dtype=torch.int64, device=gen.device)
    # a token each, and what is left of the step spread unevenly: over all of them, or over a tenth
    share = torch.rand((b,), generator=gen, device=gen.device).pow(3) + 1e-3
    if case["q"] == "mixed":
        share *= (torch.rand((b,), generator=gen, device=gen.device) < 0.1) + 1e-6
    extra = max(0, tokens - b)
    return 1 + torch.floor(share / share.sum() * (0.999 * extra)).long()


def prepare(case, seed):
    gen = torch.Generator(device=_dev()).manual_seed(int(seed))
    kind, st = case["kind"], dict(case)
    if kind == "maps":
        b, page = case["b"], case["page"]
        q = _query_lens(case, gen)
        past = torch.randint(0, case["past"] + 1, (b,), generator=gen, device=gen.device)
        width = _up(case["past"] + {"one": 1, "five": 5}.get(case["q"], case["tokens"]), page) + 2
        held = (past + page - 1) // page
        ids = torch.randperm(b * width, generator=gen, device=gen.device).to(torch.int32)
        table = ids.view(b, width).clone()
        empty = torch.arange(width, device=gen.device)[None] >= held[:, None]
        st["free"] = table[empty].contiguous()
        table[empty] = -1
        st["table"], st["head"] = table, torch.zeros((1,), dtype=torch.int32, device=gen.device)
        st["q_lens"], st["past_lens"] = q.to(torch.int32), past.to(torch.int32)
        return st
    d, hkv, page = case["d"], case["hkv"], case["page"]
    if kind == "attn":
        b, q, longest = case["b"], case["q"], case["longest"]
        lens = torch.full((b,), longest, dtype=torch.int64, device=gen.device)
        if case["ragged"]:
            lens = torch.exp(torch.rand((b,), generator=gen, device=gen.device) * math.log(longest)).round().long()
            lens = lens.clamp(min(q, longest), longest)
            lens[0] = longest
        width = _up(longest, page)
        held = ((lens + page - 1) // page)
        pages = int(held.sum()) + 1
        order = torch.randperm(pages, generator=gen, device=gen.device).to(torch.int32)
        table = torch.zeros((b, width), dtype=torch.int32, device=gen.device)
        used = torch.arange(width, device=gen.device)[None] < held[:, None]
        table[used] = order[:int(held.sum())]
        cache = _empty_cache(pages, page, hkv, d)
        bias = _heads(gen, 1, hkv, d).float()[0, :, None, :]
        step = max(1, (1 << 25) // (hkv * page * d))
        for p0 in range(0, pages, step):
            n = min(step, pages - p0)
            for i in range(2):
                x = torch.randn((n, hkv, page, d), generator=gen, device=gen.device)
                if i == 0:
                    x = x + 0.5 * bias
                codes, scale = _plain_quantize(x.to(torch.bfloat16))
                cache[i][p0:p0 + n], cache[2 + i][p0:p0 + n] = codes, scale
        st.update(cache=cache, table=table, lens=lens.to(torch.int32), lens_host=lens.tolist(), scale=d ** -0.5)
        st["query"] = torch.randn((b * q, case["h"], d), generator=gen, device=gen.device).mul_(1.5).to(torch.bfloat16)
        return st
    t = case["t"]
    pages = _up(t, page) + 2
    if kind == "cache":
        st["k"], st["v"] = _heads(gen, t, hkv, d), _heads(gen, t, hkv, d)
        st["cache"], st["slots"] = _empty_cache(pages, page, hkv, d), _slots(gen, t, page, pages)
        st["kept"] = torch.nonzero(st["slots"] >= 0)[:, 0]
        return st
    h, rot = case["h"], case["rot"]
    if case["fused_qkv"]:      # views of the merged product's rows
        qkv = _heads(gen, t, h + 2 * hkv, d)
        st["query"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    else:
        st["query"], st["k"], st["v"] = (_heads(gen, t, n, d) for n in (h, hkv, hkv))
    st["qw"] = st["kw"] = None
    if case["norm"]:
        st["qw"], st["kw"] = ((1.0 - case["offset"] + 0.2 * torch.randn((d,), generator=gen, device=gen.device))
                              .to(torch.bfloat16) for _ in range(2))
    far = 65536
    angle = torch.arange(far, device=gen.device, dtype=torch.float64)[:, None] * \
        torch.pow(1e6, -torch.arange(0, rot, 2, device=gen.device, dtype=torch.float64) / rot)[None]
    st["cos_sin"] = torch.cat((angle.cos(), angle.sin()), dim=1).to(
        torch.float32 if case["table"] == "f32" else torch.bfloat16)
    first = torch.randint(0, far - t, (1,), generator=gen, device=gen.device)
    st["positions"] = first + torch.arange(t, device=gen.device)
    st["cache"] = None
    if case["cache"]:
        st["cache"], st["slots"] = _empty_cache(pages, page, hkv, d), _slots(gen, t, page, pages)
        st["kept"] = torch.nonzero(st["slots"] >= 0)[:, 0]
    return st


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_quantize(x):
    """bf16 [..., D] -> bytes [..., D / 2] and (step, offset) bf16 [..., D / 64, 2]."""
    x = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(dim=-1), x.amax(dim=-1)
    s = ((hi - lo) / 15.0).to(torch.bfloat16)
    c = (lo - 16.0 * s.float()).to(torch.bfloat16)
    sf, cf = s.float()[..., None], c.float()[..., None]
    n = torch.where(sf == 0, 16.0, torch.round((x - cf) / sf)).clamp(16.0, 31.0) - 16.0
    n = n.to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.stack((s, c), dim=-1)


def _plain_values(codes, scale):
    """fp32 [..., D]: the bf16 values that bytes and (step, offset) stand for."""
    n = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    v = (n + 16.0) * scale[..., 0:1].float() + scale[..., 1:2].float()
    return v.to(torch.bfloat16).float().flatten(-2)


def _plain_write(k, v, slots, kept, cache):
    """Writes the tokens of the index ``kept``, those whose slot is not negative."""
    page = cache[0].shape[2]
    at, off = slots[kept] // page, slots[kept] % page
    for x, codes, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        codes[at, :, off], scale[at, :, off] = _plain_quantize(x[kept])


def _plain_read(cache, slots):
    page = cache[0].shape[2]
    kept = (slots >= 0)[:, None, None]
    at, off = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    return tuple(torch.where(kept, _plain_values(codes[at, :, off], scale[at, :, off]), 0.0).to(torch.bfloat16)
                 for codes, scale in ((cache[0], cache[2]), (cache[1], cache[3])))


def _plain_norm_rope(x, weight, st):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * (weight.float() + st["offset"])
    rot, row = st["rot"], st["cos_sin"][st["positions"]].float()[:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:]
    if st["inter"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1).to(torch.bfloat16)


def _plain_maps(st):
    page, tokens, table, free = st["page"], st["tokens"], st["table"], st["free"]
    width, dev = table.shape[1], table.device
    q, past = st["q_lens"].long().clamp(min=0), st["past_lens"].long().clamp(min=0)
    seq = past + q
    start = torch.cat((torch.zeros((1,), dtype=torch.int64, device=dev), q.cumsum(0)))
    old, new = (((n + page - 1) // page).clamp(max=width) for n in (past, seq))
    taken = new - old
    first = st["head"].long() + taken.cumsum(0) - taken
    col = torch.arange(width, device=dev)[None]
    at = first[:, None] + col - old[:, None]
    fresh = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((col >= old[:, None]) & (col < new[:, None]), fresh, table))
    ends = torch.zeros((tokens + 1,), dtype=torch.int64, device=dev)
    ends.index_add_(0, start[1:].clamp(max=tokens), torch.ones_like(q))
    i = torch.arange(tokens, device=dev)
    req = ends.cumsum(0)[:tokens].clamp(max=q.numel() - 1)
    real = i < start[-1]
    pos = past[req] + i - start[req]
    col = pos // page
    entry = table[req, col.clamp(max=width - 1)].long()
    slots = torch.where(real & (col < width) & (entry >= 0), entry * page + pos % page, -1)
    head = (st["head"].long() + taken.sum()).to(torch.int32)
    return start.to(torch.int32), seq.to(torch.int32), torch.where(real, pos, 0), slots, head, table


def _plain_attention(st):
    b, q, hkv, d = st["b"], st["q"], st["hkv"], st["d"]
    page, table, (k4, v4, ks, vs) = st["page"], st["table"], st["cache"]
    g = st["h"] // hkv
    query = st["query"].float().view(b, q, hkv, g, d)
    out = torch.zeros((b, q, hkv, g, d), device=query.device)
    for r in range(b):
        # a request's pages as [heads, keys, D]
        n = st["lens_host"][r]
        if n == 0:
            continue
        at = table[r, :_up(n, page)].long()

        def rows(codes, scale):
            return _plain_values(codes[at], scale[at]).transpose(0, 1).flatten(1, 2)[:, :n]

        keys, values = rows(k4, ks), rows(v4, vs)
        x = torch.einsum("qhgd,hnd->hqgn", query[r], keys) * st["scale"]
        last = n - q + torch.arange(q, device=x.device)
        seen = torch.arange(n, device=x.device)[None] <= last[:, None]
        x = x.masked_fill(~seen[None, :, None, :], float("-inf"))
        top = x.amax(dim=-1, keepdim=True)
        p = torch.where(seen[None, :, None, :], torch.exp(x - top), 0.0)
        total = p.sum(dim=-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        out[r] = torch.einsum("hqgn,hnd->qhgd", p, values)
    return out.view(b * q, st["h"], d).to(torch.bfloat16)


def run(st):
    kind = st["kind"]
    if own:
        if kind == "maps":
            from qwen_a100_fastpath_b200.paged import step_maps
            m = step_maps(st["q_lens"], st["past_lens"], st["table"], st["page"], st["tokens"], free_pages=st["free"],
                          free_head=st["head"])
            return m.query_start, m.seq_lens, m.positions, m.slots, m.free_head, st["table"]
        from qwen_a100_fastpath_b200.kv4 import KV4Cache, kv4_attention, kv4_read, kv4_write
        if kind == "attn":
            return kv4_attention(st["query"], KV4Cache(*st["cache"]), st["lens"], st["table"], st["q"], st["scale"])
        if kind == "cache":
            cache = KV4Cache(*st["cache"])
            kv4_write(st["k"], st["v"], st["slots"], cache)
            return kv4_read(cache, st["slots"])
        from qwen_a100_fastpath_b200.norms import qk_norm_rope
        kw = dict(eps=EPS, weight_offset=st["offset"], interleaved=st["inter"])
        if st["cache"] is None:
            return qk_norm_rope(st["query"], st["k"], st["qw"], st["kw"], st["positions"], st["cos_sin"], **kw)
        cache = KV4Cache(*st["cache"])
        query, _ = qk_norm_rope(st["query"], st["k"], st["qw"], st["kw"], st["positions"], st["cos_sin"], v=st["v"],
                                cache=cache, slots=st["slots"], **kw)
        return (query, *kv4_read(cache, st["slots"]))
    if kind == "maps":
        return _plain_maps(st)
    if kind == "attn":
        return _plain_attention(st)
    if kind == "cache":
        _plain_write(st["k"], st["v"], st["slots"], st["kept"], st["cache"])
        return _plain_read(st["cache"], st["slots"])
    query, k = (_plain_norm_rope(st[x], st[w], st) for x, w in (("query", "qw"), ("k", "kw")))
    if st["cache"] is None:
        return query, k
    _plain_write(k, st["v"], st["slots"], st["kept"], st["cache"])
    return (query, *_plain_read(st["cache"], st["slots"]))


# ------------------------------------------------------------------------------------------------ in 64 bits
def _values_64(codes, scale):
    d = torch.float64
    n = torch.empty((*codes.shape[:-1], codes.shape[-1] * 2), dtype=d, device=codes.device)
    n[..., 0::2], n[..., 1::2] = (codes % 16).to(d), (codes // 16).to(d)
    s, c = (scale[..., i].to(d).repeat_interleave(GROUP, dim=-1) for i in range(2))
    return n.add_(16.0).mul_(s).add_(c).float().to(torch.bfloat16).to(d)


def _kept_64(x):
    """What the cache keeps of the bf16 values x (given in 64 bits): step and offset are bf16 numbers."""
    out = torch.empty_like(x)
    for j in range(0, x.shape[-1], GROUP):
        part = x[..., j:j + GROUP]
        low, high = part.min(dim=-1, keepdim=True).values, part.max(dim=-1, keepdim=True).values
        s = ((high - low) / 15).float().to(torch.bfloat16).double()
        c = (low - 16 * s).float().to(torch.bfloat16).double()
        n = torch.round((part - c) / torch.where(s == 0, 1.0, s)).clamp_(16, 31)
        out[..., j:j + GROUP] = torch.where(s == 0, c, n * s + c)
    return out.float().to(torch.bfloat16).double()


def _maps_by_hand(st):
    page, tokens = st["page"], st["tokens"]
    table, free = st["table"].tolist(), st["free"].tolist()
    taken, start, seq = st["head"].item(), [0], []
    pos, slots = [0] * tokens, [-1] * tokens
    for r, (q, past) in enumerate(zip(st["q_lens"].tolist(), st["past_lens"].tolist())):
        row, n = table[r], past + q
        for p in range(min(_up(past, page), len(row)), min(_up(n, page), len(row))):
            row[p] = free[taken] if taken < len(free) else -1
            taken += 1
        for j in range(past, n):
            i = start[-1] + j - past
            if i < tokens:
                pos[i] = j
                if j // page < len(row) and row[j // page] >= 0:
                    slots[i] = row[j // page] * page + j % page
        start.append(start[-1] + q)
        seq.append(n)
    dev = st["table"].device
    return tuple(torch.tensor(x, dtype=t, device=dev) for x, t in (
        (start, torch.int32), (seq, torch.int32), (pos, torch.int64), (slots, torch.int64), ([taken], torch.int32),
        (table, torch.int32)))


def exact(case, seed):
    st = prepare(case, seed)
    kind, d64 = case["kind"], torch.float64
    if kind == "maps":
        return _maps_by_hand(st)
    if kind == "attn":
        b, q, h, hkv, page = (case[x] for x in ("b", "q", "h", "hkv", "page"))
        g, (k4, v4, ks, vs) = h // hkv, st["cache"]
        out = torch.zeros((b, q, h, case["d"]), dtype=d64, device=k4.device)
        query = st["query"].to(d64).view(b, q, h, case["d"])
        for r, n in enumerate(st["lens"].tolist()):
            at = st["table"][r, torch.arange(n, device=k4.device) // page].long()
            off = torch.arange(n, device=k4.device) % page
            for j in range(hkv if n else 0):
                keys, values = _values_64(k4[at, j, off], ks[at, j, off]), _values_64(v4[at, j, off], vs[at, j, off])
                for i in range(q):
                    m = n - q + i + 1
                    if m > 0:
                        w = torch.softmax(query[r, i, j * g:(j + 1) * g] @ keys[:m].t() * st["scale"], dim=1)
                        out[r, i, j * g:(j + 1) * g] = w @ values[:m]
        return out.view(b * q, h, case["d"])
    if kind == "cache":
        kept = (st["slots"] >= 0)[:, None, None]
        return tuple(torch.where(kept, _kept_64(st[x].to(d64)), 0.0) for x in ("k", "v"))

    def turned(x, w):
        x = x.to(d64)
        if w is not None:
            x = x / (x.square().sum(dim=-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (w.to(d64) + case["offset"])
        rot = case["rot"]
        first = torch.arange(0, rot, 2, device=x.device) if case["inter"] else torch.arange(rot // 2, device=x.device)
        second = first + (1 if case["inter"] else rot // 2)
        row = st["cos_sin"].to(d64)[st["positions"]].unsqueeze(1)
        y = x.clone()
        y[..., first] = x[..., first] * row[..., :rot // 2] - x[..., second] * row[..., rot // 2:]
        y[..., second] = x[..., second] * row[..., :rot // 2] + x[..., first] * row[..., rot // 2:]
        return y

    query, k = turned(st["query"], st["qw"]), turned(st["k"], st["kw"])
    if not case["cache"]:
        return query, k
    kept = (st["slots"] >= 0)[:, None, None]
    # the rotated keys are bf16 before they are kept, so that a rounding there may move one to the next step
    return query, None, torch.where(kept, _kept_64(st["v"].to(d64)), 0.0)


def work(case):
    kind = case["kind"]
    if kind == "maps":
        b, t = case["b"], case["tokens"]
        # lengths and starts of each request, position and slot of each token, an entry of the table for each page met
        return {"bytes": 16 * b + 16 * t + 8 * (_up(t, case["page"]) + b), "flops": 8 * t}
    d, hkv = case["d"], case["hkv"]
    if kind == "attn":
        b, q, h, n = case["b"], case["q"], case["h"], case["longest"]
        if case["ragged"] and b > 1 and n > 1:    # the mean of lengths spread evenly over their logarithm
            n = (n + (b - 1) * (n - 1) / math.log(n)) / b
        return {"bytes": int(2 * b * n * hkv * (d // 2 + d // 16)) + 4 * b * q * h * d, "flops": int(4 * b * q * h * n * d)}
    t = case["t"]
    kept = 2 * t * hkv * (d // 2 + d // 16)     # written, or read back
    if kind == "cache":
        return {"bytes": 2 * kept + 8 * t * hkv * d + 8 * t, "flops": 12 * t * hkv * d}
    h, table = case["h"], 4 if case["table"] == "f32" else 2
    read = 2 * t * (h + hkv) * d + t * (8 + table * case["rot"])
    if not case["cache"]:
        return {"bytes": read + 2 * t * (h + hkv) * d, "flops": 10 * t * (h + hkv) * d}
    return {"bytes": read + 2 * t * (h + hkv) * d + 2 * kept + 4 * t * hkv * d + 8 * t,
            "flops": 10 * t * (h + 2 * hkv) * d}
