"""The block-scaled fp8 linear path of a decoder layer, as measured: the matrix product of e4m3 operands with one scale
for each 128 elements along k (and each 128 output channels of the weight), the activation quantizer in front of it
(alone, or behind the MLP's SiLU gate), the two as one linear layer on bf16 activations, and the residual update with
the norms on both sides of a block.

``run`` computes them in elementary torch operations where ``own`` is false, and through this package's public entry
points where it is true.  Sizes are this repository's decoder layer (hidden 5120, qkv 10240, attention output 8192,
gate_up 34816, MLP 17408) and, in ``draw``, everything around it.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = E4M3_MAX * 2.0 ** -60   # an all-zero group gets the scale 2^-60 and zeros
ACTS = ("none", "sigmoid", "silu")


def listed():
    return [
        # o_proj of one token: the smallest product, bound by its launch and 42 MB of weights
        dict(name="mm_token", kind="mm", m=1, n=5120, k=8192, bias=False, out="bf16"),
        # gate_up of a verification batch (one token and four drafts)
        dict(name="mm_verify", kind="mm", m=5, n=34816, k=5120, bias=False, out="bf16"),
        # qkv of a batch of decoding requests, above the single-tile sizes
        dict(name="mm_batch", kind="mm", m=72, n=10240, k=5120, bias=False, out="bf16"),
        # a ragged product: no size a multiple of a tile, a bias, an fp32 result (a router or a small head)
        dict(name="mm_ragged", kind="mm", m=333, n=2600, k=1160, bias=True, out="f32"),
        # gate_up of a whole prompt: the largest product, bound by the tensor cores
        dict(name="mm_prefill", kind="mm", m=4096, n=34816, k=5120, bias=False, out="bf16"),
        # down of one token, from bf16 activations
        dict(name="linear_token", kind="linear", m=1, n=5120, k=17408, bias=False),
        # qkv of sixteen tokens with its bias, from bf16 activations
        dict(name="linear_verify", kind="linear", m=16, n=10240, k=5120, bias=True),
        # o_proj of a prompt chunk, from bf16 activations
        dict(name="linear_prefill", kind="linear", m=2048, n=5120, k=8192, bias=False),
        # the MLP activation of a verification batch, quantized for down
        dict(name="quant_gate_verify", kind="quant", m=5, k=17408, silu_mul=True),
        # the same for a prompt
        dict(name="quant_gate_prefill", kind="quant", m=4096, k=17408, silu_mul=True),
        # attention norm of one token with the residual update in front, quantized for qkv
        dict(name="norm_token", kind="norm", m=1, h=5120, post=False, gate="none", act="none", residual="bf16",
             alpha=1.0, offset=0.0, quantize=True),
        # norms on both sides of a gated block over a prompt, fp32 residual stream with a residual scale
        dict(name="norm_prefill", kind="norm", m=8192, h=5120, post=True, gate="full", act="sigmoid", residual="f32",
             alpha=0.7, offset=1.0, quantize=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size between lo and hi over its logarithm: half of them multiples of 128, a quarter of 8, a quarter any."""
    v = _log_int(rng, lo, hi)
    r = rng.random()
    step = 128 if r < 0.5 else 8 if r < 0.75 else 1
    return max(step, v // step * step)


def draw(rng):
    kind = rng.choice(("mm", "mm", "linear", "quant", "norm"))
    if kind in ("mm", "linear"):
        m = _log_int(rng, 1, 4096)
        n = _size(rng, 64, 34816)
        k = _size(rng, 128, 17408)
        while m * n * k > 4096 * 34816 * 5120:
            m = max(1, m // 2)
        case = dict(kind=kind, m=m, n=n, k=k, bias=rng.random() < 0.4)
        if kind == "mm":
            case["out"] = rng.choice(("bf16", "bf16", "f32"))
        return case
    if kind == "quant":
        return dict(kind="quant", m=_log_int(rng, 1, 4096), k=_size(rng, 128, 17408), silu_mul=rng.random() < 0.5)
    gate = rng.choice(("none", "full", "channel", "token"))
    return dict(kind="norm", m=_log_int(rng, 1, 8192), h=_size(rng, 128, 8192), post=rng.random() < 0.5, gate=gate,
                act=rng.choice(ACTS) if gate != "none" else "none", residual=rng.choice(("bf16", "f32")),
                alpha=rng.choice((1.0, 0.7, 0.22)), offset=rng.choice((0.0, 1.0)), quantize=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _activations(gen, m, k):
    """Hidden states: normal values, a spread of channel sizes, a few outlier channels twenty times the others'."""
    x = torch.randn((m, k), generator=gen, device=gen.device)
    x *= torch.exp(0.5 * torch.randn((k,), generator=gen, device=gen.device))
    loud = torch.rand((k,), generator=gen, device=gen.device) < 0.002
    return (x * torch.where(loud, 20.0, 1.0)).to(torch.bfloat16)


def _weight(gen, n, k):
    """A checkpoint's weight: e4m3 rows of 16-byte stride and one scale for each block of 128 x 128, as loaded."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros((nb * BLOCK, kb * BLOCK), device=gen.device)
    w[:n, :k] = 0.02 * torch.randn((n, k), generator=gen, device=gen.device)
    w[:n] *= torch.exp(0.3 * torch.randn((n, 1), generator=gen, device=gen.device))
    blocks = w.view(nb, BLOCK, kb, BLOCK)
    scale = blocks.abs().amax(dim=(1, 3)).clamp_(min=1e-12) / E4M3_MAX
    blocks /= scale[:, None, :, None]
    rows = torch.zeros((n, -(-k // 16) * 16), dtype=torch.float8_e4m3fn, device=gen.device)
    rows[:, :k] = w[:n, :k].clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return rows[:, :k].t(), scale


def _quantized(x):
    """Activations of the product as the quantizer leaves them: e4m3 rows of 16-byte stride, fp32 scales."""
    q, scale = _plain_quantize(x.float())
    m, k = x.shape
    rows = torch.zeros((m, -(-k // 16) * 16), dtype=torch.float8_e4m3fn, device=x.device)
    rows[:, :k] = q
    return rows[:, :k], scale


def prepare(case, seed):
    gen = torch.Generator(device=_dev()).manual_seed(int(seed))
    m, kind = case["m"], case["kind"]
    st = dict(case)
    if kind in ("mm", "linear"):
        n, k = case["n"], case["k"]
        x = _activations(gen, m, k)
        if kind == "mm":
            st["a"], st["a_scale"] = _quantized(x)
        else:
            st["x"] = x
        st["w_t"], st["w_scale"] = _weight(gen, n, k)
        st["b"] = (0.1 * torch.randn((n,), generator=gen, device=gen.device)).to(torch.bfloat16) if case["bias"] else None
    elif kind == "quant":
        st["x"] = _activations(gen, m, 2 * case["k"] if case["silu_mul"] else case["k"])
    else:
        h = case["h"]
        st["x"] = _activations(gen, m, h)
        r = 3.0 * _activations(gen, m, h).float()
        st["r"] = r if case["residual"] == "f32" else r.to(torch.bfloat16)

        def gamma():
            return (1.0 - case["offset"] + 0.2 * torch.randn((h,), generator=gen, device=gen.device)).to(torch.bfloat16)

        st["pre"] = gamma()
        st["post_w"] = gamma() if case["post"] else None
        shape = {"none": None, "full": (m, h), "channel": (h,), "token": (m, 1)}[case["gate"]]
        st["g"] = None if shape is None else (1.5 * torch.randn(shape, generator=gen, device=gen.device)).to(torch.bfloat16)
    return st


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_quantize(x):
    """fp32 [m, k] -> e4m3 [m, k] and the fp32 scale of each group of 128 along k."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    padded = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    amax = padded.abs().amax(dim=2).clamp(min=AMAX_FLOOR)
    q = (padded * (E4M3_MAX / amax)[:, :, None]).view(m, kb * BLOCK)[:, :k]
    return q.to(torch.float8_e4m3fn), amax / E4M3_MAX


def _plain_mm(a, a_scale, w_t, w_scale, bias):
    """fp32 result of the block-scaled product: both operands scaled to fp32, one product."""
    k, n = w_t.shape
    af = a.float() * a_scale.repeat_interleave(BLOCK, dim=1)[:, :k]
    wf = w_t.t().float() * w_scale.repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    y = af @ wf.t()
    return y if bias is None else y + bias.float()


def _plain_act(g, act):
    g = g.float()
    if act == "none":
        return g
    s = 1.0 / (1.0 + torch.exp(-g))
    return s if act == "sigmoid" else g * s


def _plain_rms(x, weight, offset, eps):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + eps) * (weight.float() + offset)


EPS = 1e-6


def run(st):
    kind = st["kind"]
    if own:
        if kind == "mm":
            from qwen_a100_fastpath_b200.fp8 import fp8_block_mm
            return fp8_block_mm(st["a"], st["a_scale"], st["w_t"], st["w_scale"], bias=st["b"],
                                out_dtype=torch.float32 if st["out"] == "f32" else torch.bfloat16)
        if kind == "linear":
            from qwen_a100_fastpath_b200.fp8 import fp8_block_linear
            return fp8_block_linear(st["x"], st["w_t"], st["w_scale"], bias=st["b"])
        if kind == "quant":
            from qwen_a100_fastpath_b200.fp8 import fp8_quantize
            return fp8_quantize(st["x"], silu_mul=st["silu_mul"])
        from qwen_a100_fastpath_b200.norms import residual_norm
        return residual_norm(st["x"], st["r"], st["pre"], eps=EPS, post_weight=st["post_w"], gate=st["g"],
                             gate_act=st["act"], residual_scale=st["alpha"], weight_offset=st["offset"],
                             quantize=st["quantize"])
    if kind == "mm":
        y = _plain_mm(st["a"], st["a_scale"], st["w_t"], st["w_scale"], st["b"])
        return y if st["out"] == "f32" else y.to(torch.bfloat16)
    if kind == "linear":
        q, scale = _plain_quantize(st["x"].float())
        return _plain_mm(q, scale, st["w_t"], st["w_scale"], st["b"]).to(torch.bfloat16)
    if kind == "quant":
        x = st["x"].float()
        if st["silu_mul"]:
            g, u = x[:, :st["k"]], x[:, st["k"]:]
            x = g / (1.0 + torch.exp(-g)) * u
        return _plain_quantize(x)
    v = st["x"].float()
    if st["post"]:
        v = _plain_rms(v, st["post_w"], st["offset"], EPS)
    if st["g"] is not None:
        v = v * _plain_act(st["g"], st["act"])
    r = st["r"].float() + st["alpha"] * v
    h = _plain_rms(r, st["pre"], st["offset"], EPS)
    h = _plain_quantize(h) if st["quantize"] else h.to(torch.bfloat16)
    return h, r.to(st["r"].dtype)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _e4m3_64(v):
    """Nearest e4m3 value, ties to even: three mantissa bits down to 2^-6, steps of 2^-9 below, at most 448."""
    _, e = torch.frexp(v)                       # |v| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _groups_64(x):
    """(e4m3 values, scales) of 64-bit rows; the scale is the fp32 number that is kept."""
    q, s = torch.empty_like(x), []
    for c in range(0, x.shape[1], BLOCK):
        part = x[:, c:c + BLOCK]
        top = part.abs().max(dim=1).values.clamp(min=448.0 * 2.0 ** -60)
        q[:, c:c + BLOCK] = _e4m3_64(part * (448.0 / top)[:, None])
        s.append(top / 448.0)
    return q, torch.stack(s, dim=1)


def exact(case, seed):
    st = prepare(case, seed)
    kind, d = case["kind"], torch.float64
    if kind in ("mm", "linear"):
        if kind == "mm":
            q, s = st["a"].to(d), st["a_scale"].to(d)
        else:
            q, s = _groups_64(st["x"].to(d))
            s = s.float().to(d)
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros((m, n), dtype=d, device=q.device)
        rows = torch.arange(n, device=q.device) // BLOCK
        for g in range(-(-k // BLOCK)):
            c = slice(g * BLOCK, min(k, (g + 1) * BLOCK))
            y += (q[:, c] @ st["w_t"][c].to(d)) * s[:, g, None] * st["w_scale"].to(d)[rows, g][None, :]
        return y if st["b"] is None else y + st["b"].to(d)
    if kind == "quant":
        x = st["x"].to(d)
        if case["silu_mul"]:
            x = x[:, :case["k"]] * torch.sigmoid(x[:, :case["k"]]) * x[:, case["k"]:]
        return _groups_64(x)

    def rms(t, w):
        return t / (t.square().sum(dim=1, keepdim=True) / t.shape[1] + EPS).sqrt() * (w.to(d) + case["offset"])

    v = st["x"].to(d)
    if case["post"]:
        v = rms(v, st["post_w"])
    if st["g"] is not None:
        g = st["g"].to(d)
        v = v * {"none": g, "sigmoid": torch.sigmoid(g), "silu": g * torch.sigmoid(g)}[case["act"]]
    r = st["r"].to(d) + case["alpha"] * v
    h = rms(r, st["pre"])
    return _groups_64(h) if case["quantize"] else h, r


def work(case):
    m, kind = case["m"], case["kind"]

    def blocks(v):
        return -(-v // BLOCK)

    if kind in ("mm", "linear"):
        n, k = case["n"], case["k"]
        x = 2 * m * k if kind == "linear" else m * k + 4 * m * blocks(k)
        out = 4 if case.get("out") == "f32" else 2
        return {"bytes": x + n * k + 4 * blocks(n) * blocks(k) + (2 * n if case["bias"] else 0) + out * m * n,
                "flops": 2 * m * n * k}
    if kind == "quant":
        k = case["k"]
        return {"bytes": (4 if case["silu_mul"] else 2) * m * k + m * k + 4 * m * blocks(k),
                "flops": (8 if case["silu_mul"] else 3) * m * k}
    h = case["h"]
    gate = {"none": 0, "full": m * h, "channel": h, "token": m}[case["gate"]]
    r = 4 if case["residual"] == "f32" else 2
    out = m * h + 4 * m * blocks(h) if case["quantize"] else 2 * m * h
    return {"bytes": 2 * m * h + 2 * r * m * h + 2 * gate + 2 * h * (2 if case["post"] else 1) + out,
            "flops": 12 * m * h}
