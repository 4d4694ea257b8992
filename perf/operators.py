"""The microscaled 4-bit (MX4) operators: what is timed and compared.

MX4 is the OCP microscaling format MXFP4: 4-bit floats e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives) in blocks of 32, each block with one power-of-two scale E8M0 (a byte E, value
2^(E - 127), 255 = NaN). A block of amplitude a gets the scale 2^(floor(log2 a) - 2); the values
are rounded to nearest, ties to the even code, and saturate at 6. Before it is quantized a row
may be rotated by the regular Hadamard matrix in groups of 16, 64 or 256 (0: not rotated).

Four operators:

* ``quantize``: rows to MX4 and back to the values the codes stand for.
* ``linear``: rows quantized to MX4, times a weight already held in MX4, plus bias.
* ``cache``: new keys and values written to a paged MX4 cache, then a list of slots read back.
* ``attention``: queries of the newest tokens against a paged MX4 cache.

Layouts. Codes: two a byte, the even column in the low nibble. Scales of a matrix [R, K]:
[ceil(R/128), ceil(K/128), 512], the byte of row r and block b at (r % 32) * 16 + (r / 32 % 4) * 4
+ b % 4 of tile (r / 128, b / 4). Cache: codes [pages, 2, heads, page, D/2] and scales
[pages, 2, heads, page, D/32], keys at index 0 and values at 1, both rotated along D.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    """This repository's package (its folder's name is no module name)."""
    at = os.path.join(HERE, "comfyui-int4-convrot-rdna4_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import _int4
    return _int4


# ---------------------------------------------------------------- the cases


def listed():
    return [
        # one new token's hidden state ahead of a projection: latency only
        {"name": "quantize_one_token", "op": "quantize", "rows": 1, "k": 3840, "group": 256, "dtype": "bf16"},
        # text embeddings of a prompt, an odd count of tokens, half precision
        {"name": "quantize_text", "op": "quantize", "rows": 509, "k": 4096, "group": 64, "dtype": "f16"},
        # the MLP's inner activations of a 1024 x 1024 image and its text at hidden 3840
        {"name": "quantize_image", "op": "quantize", "rows": 4608, "k": 15360, "group": 256, "dtype": "bf16"},
        # a projection for a single decoded token: the weight's bytes
        {"name": "linear_one_token", "op": "linear", "m": 1, "n": 15360, "k": 3840, "group": 256, "bias": True, "dtype": "bf16"},
        # a short prompt (odd count) through the MLP's down projection
        {"name": "linear_text", "op": "linear", "m": 333, "n": 3840, "k": 15360, "group": 256, "bias": True, "dtype": "f16"},
        # image tokens of the largest size of the token sweep through the MLP's up projection
        {"name": "linear_image", "op": "linear", "m": 16384, "n": 15360, "k": 3840, "group": 256, "bias": True, "dtype": "bf16"},
        # one decode step of a small batch: a token each is written, one short sequence is read back
        {"name": "cache_decode", "op": "cache", "new": 7, "read": 129, "heads": 8, "d": 128, "page": 16, "group": 64, "dtype": "bf16"},
        # a chunk of a prefill: the chunk is written, the context so far is read for it
        {"name": "cache_chunk", "op": "cache", "new": 2047, "read": 8191, "heads": 8, "d": 64, "page": 32, "group": 16, "dtype": "f16"},
        # several long prompts at once
        {"name": "cache_prompts", "op": "cache", "new": 32768, "read": 65536, "heads": 8, "d": 128, "page": 64, "group": 64, "dtype": "bf16"},
        # one user's short conversation, one token
        {"name": "attention_short", "op": "attention", "b": 1, "tq": 1, "hq": 32, "hkv": 8, "d": 128, "page": 64, "group": 64,
         "longest": 777, "ragged": False, "dtype": "bf16"},
        # a ragged batch with empty slots, three drafted tokens to verify besides the last one
        {"name": "attention_drafts", "op": "attention", "b": 37, "tq": 4, "hq": 24, "hkv": 8, "d": 64, "page": 16, "group": 64,
         "longest": 4096, "ragged": True, "dtype": "f16"},
        # long contexts, one token each: the cache's bytes
        {"name": "attention_long", "op": "attention", "b": 16, "tq": 1, "hq": 64, "hkv": 8, "d": 128, "page": 64, "group": 64,
         "longest": 32768, "ragged": False, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "cache", "attention"))
    if op in ("quantize", "linear"):
        group = rng.choice((0, 16, 64, 256))
        unit = max(group, BLOCK)
        k = unit * _between(rng, max(1, 512 // unit), 15360 // unit)
        if op == "quantize":
            rows = _between(rng, 1, min(16384, 4608 * 15360 // k))
            return {"op": op, "rows": rows, "k": k, "group": group, "dtype": rng.choice(("bf16", "f16", "f32"))}
        m = _between(rng, 1, 16384)
        n = _between(rng, 64, min(15360, 16384 * 15360 * 3840 // (m * k)))
        return {"op": op, "m": m, "n": n, "k": k, "group": group, "bias": rng.random() < 0.7, "dtype": rng.choice(("bf16", "f16"))}
    d = rng.choice((64, 128, 256))
    group = rng.choice((0, 16, 64))
    page = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("bf16", "f16"))
    hkv = rng.choice((1, 2, 4, 8, 16))
    if op == "cache":
        new = _between(rng, 1, 32768 * 8 * 128 // (hkv * d) if hkv * d > 1024 else 32768)
        read = _between(rng, 1, 65536 * 8 * 128 // (hkv * d) if hkv * d > 1024 else 65536)
        return {"op": op, "new": new, "read": read, "heads": hkv, "d": d, "page": page, "group": group, "dtype": dtype}
    b = _between(rng, 1, 128)
    longest = _between(rng, 1, min(131072, 16 * 32768 * 8 * 128 // (b * hkv * d)))
    return {"op": op, "b": b, "tq": rng.choice((1, 1, 2, 3, 4, 8)), "hq": hkv * rng.choice((1, 2, 3, 4, 8)), "hkv": hkv, "d": d, "page": page,
            "group": group, "longest": longest, "ragged": rng.random() < 0.7, "dtype": dtype}


def _lengths(case, seed):
    """The sequences' lengths: host data that a scheduler has. Ragged batches hold an empty one, one of one token and the longest."""
    b, longest = case["b"], case["longest"]
    if not case["ragged"]:
        return [longest] * b
    import random
    rng = random.Random(1000003 * seed + b)
    return [(longest, 0, 1)[i] if i < 3 else rng.randint(0, longest) for i in range(b)]


def work(case):
    op = case["op"]
    if op == "quantize":
        n, size = case["rows"] * case["k"], DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (size + 2), "flops": n}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * 17 / 32 + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "cache":
        values = 2 * case["heads"] * case["d"]
        return {"bytes": case["new"] * (values * (2 + 17 / 32) + 8) + case["read"] * (values * (2 + 17 / 32) + 8),
                "flops": (case["new"] + case["read"]) * values}
    # the lengths of a ragged batch go by the seed: half the longest on average
    b = case["b"]
    tokens = b * case["longest"] if not case["ragged"] else case["longest"] * (1 if b < 3 else 1 + max(0, b - 3) / 2)
    rows = case["tq"] * case["hq"]
    return {"bytes": tokens * case["hkv"] * case["d"] * 2 * 17 / 32 + 2 * 2 * b * rows * case["d"], "flops": 4 * tokens * rows * case["d"]}


# ---------------------------------------------------------------- plain forms (32 bits, elementary operations)


def _h4(v, dim):
    """out_i = (v0 + v1) + (v2 + v3) - 2 v_(3-i) along a dimension of four."""
    v0, v1, v2, v3 = v.unbind(dim)
    s = (v0 + v1) + (v2 + v3)
    return torch.stack((s - 2 * v3, s - 2 * v2, s - 2 * v1, s - 2 * v0), dim)


def _rotate(x, group):
    """x [..., K] (32 bits) by the regular Hadamard matrix in groups; symmetric, so this is its inverse too."""
    if not group:
        return x
    shape = x.shape
    if group == 16:
        v = x.reshape(-1, 4, 4)
        v = _h4(_h4(v, 2), 1)
    elif group == 64:
        v = x.reshape(-1, 4, 4, 4)
        v = _h4(_h4(_h4(v, 3), 2), 1)
    else:
        v = x.reshape(-1, 4, 4, 4, 4)
        v = _h4(_h4(_h4(_h4(v, 4), 3), 2), 1)
    return (v * (1 / math.sqrt(group))).reshape(shape)


def _encode(x):
    """x [..., K] (32 bits) to codes 0..15 [..., K] and scale bytes [..., K/32]."""
    v = x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    a = v.abs().amax(-1)
    bad = ~torch.isfinite(a)
    e = (torch.frexp(torch.where(bad, 1.0, a))[1] - 1 - 2).clamp(-127, 125)
    e = torch.where(a == 0, -127, e)
    y = torch.ldexp(v, -e.unsqueeze(-1))
    m = y.abs()
    c = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8) + (m >= 1.75).to(torch.uint8)
         + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8) + (m > 5).to(torch.uint8))
    c = c | (torch.signbit(y).to(torch.uint8) << 3)
    return c.reshape(x.shape), torch.where(bad, 255, e + 127).to(torch.uint8)


def _values(codes, scales):
    """Codes 0..15 [..., K] and scale bytes [..., K/32] as the numbers they stand for, in 32 bits."""
    table = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    v = table[codes.int()].reshape(*scales.shape, BLOCK)
    e = scales.to(torch.int32).unsqueeze(-1)
    return torch.where(e == 255, math.nan, torch.ldexp(v, e - 127)).reshape(codes.shape)


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], packed.shape[-1] * 2)


def _tile(scales):
    """Scale bytes [R, K/32] in tiles of 128 rows and 4 blocks."""
    r, b = scales.shape
    rt, kt = -(-r // 128), -(-b // 4)
    full = scales.new_zeros(rt * 128, kt * 4)
    full[:r, :b] = scales
    return full.reshape(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512)


def _untile(tiles, r, b):
    rt, kt, _ = tiles.shape
    return tiles.reshape(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:r, :b]


def _plain_quantize(s):
    c, e = _encode(_rotate(s["x"].float(), s["group"]))
    return _values(c, e).to(torch.bfloat16)


def _plain_linear(s):
    x = s["x"]
    c, e = _encode(_rotate(x.float(), s["group"]))
    w = _values(_unpack(s["weight"]), _untile(s["wscales"], s["weight"].shape[0], x.shape[1] // BLOCK))
    out = _values(c, e) @ w.t()
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(x.dtype)


def _plain_cache(s):
    page = s["codes"].shape[3]
    to, off = s["write"] // page, s["write"] % page
    for i, new in enumerate((s["k"], s["v"])):
        c, e = _encode(_rotate(new.float(), s["group"]))
        s["codes"][to, i, :, off] = _pack(c)
        s["scales"][to, i, :, off] = e
    at, off = s["read"] // page, s["read"] % page
    return tuple(_rotate(_values(_unpack(s["codes"][at, i, :, off]), s["scales"][at, i, :, off]), s["group"]).to(s["k"].dtype) for i in (0, 1))


def _plain_attention(s):
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    b, tq, hq, d = q.shape
    _, _, hkv, page, _ = s["codes"].shape
    n = table.shape[1] * page
    qr = _rotate(q.float(), s["group"]).reshape(b, tq, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)

    def gathered(i):
        c, e = s["codes"][table, i], s["scales"][table, i]                       # [b, pages, heads, page, .]
        return _values(_unpack(c), e).transpose(1, 2).reshape(b, hkv, n, d)

    at = torch.arange(n, device=q.device)
    last = (lens[:, None] - tq + torch.arange(tq, device=q.device)).repeat_interleave(hq // hkv, 1)    # newest position a row sees
    seen = at[None, None, None, :] <= last[:, None, :, None]
    score = (qr @ gathered(0).transpose(2, 3)) * s["scale"]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = _rotate(p @ gathered(1), s["group"])
    return out.reshape(b, hkv, tq, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, tq, hq, d).to(q.dtype)


# ---------------------------------------------------------------- inputs


def _activations(rows, k, dtype, g):
    """N(0, 1) with one channel of a hundred twenty times larger, as the models' hidden states are."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    at = torch.randperm(k, generator=g, device="cuda")[: max(1, k // 100)]
    x[:, at] *= 20
    return x.to(DTYPES[dtype])


def _cache(pages, heads, page, d, group, g):
    """A cache that holds keys and values of earlier tokens in every slot."""
    codes = torch.empty(pages, 2, heads, page, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, 2, heads, page, d // BLOCK, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (2 * heads * page * d))
    for at in range(0, pages, step):
        to = min(pages, at + step)
        x = torch.randn(to - at, 2, heads, page, d, generator=g, device="cuda")
        x[..., 0, :, :, 3] *= 8                                                  # keys have channels that stand out
        c, e = _encode(_rotate(x, group))
        codes[at:to], scales[at:to] = _pack(c), e
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, group = case["op"], case["group"]
    if op == "quantize":
        return {"op": op, "group": group, "x": _activations(case["rows"], case["k"], case["dtype"], g)}
    if op == "linear":
        n, k = case["n"], case["k"]
        c, e = _encode(_rotate(torch.randn(n, k, generator=g, device="cuda") * 0.02, group))
        bias = (torch.randn(n, generator=g, device="cuda") * 0.01).to(DTYPES[case["dtype"]]) if case["bias"] else None
        return {"op": op, "group": group, "x": _activations(case["m"], k, case["dtype"], g), "weight": _pack(c), "wscales": _tile(e), "bias": bias}
    if op == "cache":
        heads, d, page, new, read = (case[n] for n in ("heads", "d", "page", "new", "read"))
        pages = -(-max(new, read) // page) + 2
        codes, scales = _cache(pages, heads, page, d, group, g)
        slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        slots = slots.reshape(-1)                                                # a sequence's tokens: page after page, the pages anywhere
        qkv = _activations(new, 3 * heads * d, case["dtype"], g).reshape(new, 3, heads, d)
        return {"op": op, "group": group, "codes": codes, "scales": scales, "k": qkv[:, 1], "v": qkv[:, 2],
                "write": slots[max(0, read - new):][:new].contiguous(), "read": slots[:read].contiguous()}
    b, tq, hq, hkv, d, page = (case[n] for n in ("b", "tq", "hq", "hkv", "d", "page"))
    lens = _lengths(case, seed)
    each = max(1, -(-case["longest"] // page))
    codes, scales = _cache(b * each, hkv, page, d, group, g)
    table = torch.randperm(b * each, generator=g, device="cuda").reshape(b, each).int()
    q = _activations(b * tq, hq * d, case["dtype"], g).reshape(b, tq, hq, d)
    q = (q.float().clamp(-4, 4)).to(q.dtype)                                      # queries are normalised ahead of attention
    return {"op": op, "group": group, "codes": codes, "scales": scales, "q": q, "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "scale": 1 / math.sqrt(d)}


def run(state):
    op, s = state["op"], state
    if not own:
        return {"quantize": _plain_quantize, "linear": _plain_linear, "cache": _plain_cache, "attention": _plain_attention}[op](s)
    mx4 = _package()
    if op == "quantize":
        codes, scales = mx4.quantize_convrot_mx4(s["x"], s["group"])
        return mx4.dequantize_convrot_mx4(codes, scales, dtype=torch.bfloat16)
    if op == "linear":
        return mx4.convrot_mx4_linear(s["x"], s["weight"], s["wscales"], s["bias"], convrot_groupsize=s["group"])
    if op == "cache":
        mx4.convrot_mx4_cache_append(s["codes"], s["scales"], s["k"], s["v"], s["write"], convrot_groupsize=s["group"])
        return mx4.convrot_mx4_cache_read(s["codes"], s["scales"], s["read"], dtype=s["k"].dtype, convrot_groupsize=s["group"])
    return mx4.convrot_mx4_attention(s["q"], s["codes"], s["scales"], s["table"], s["lens"], softmax_scale=s["scale"], convrot_groupsize=s["group"])


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_rotate(x, group):
    if not group:
        return x
    h4 = 1 - 2 * torch.eye(4, dtype=torch.float64, device=x.device).flip(0)
    h = torch.ones(1, 1, dtype=torch.float64, device=x.device)
    while h.shape[0] < group:
        h = torch.kron(h, h4 / 2)
    return (x.reshape(-1, group) @ h).reshape(x.shape)


def _exact_quantized(x):
    """The nearest values of the format to x [..., K] (64 bits), ties to the even one."""
    v = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = torch.floor(torch.log2(v.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -140)))
    unit = torch.exp2((top - 2).clamp(-127, 125))
    y = v / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1.0))) - 1)        # spacing: 0.5 below 2, then 1, then 2
    return ((torch.round(y / step) * step).clamp(-6, 6) * unit).reshape(x.shape)


def _exact_decoded(packed, scales):
    """Bytes of codes [..., K/2] and scales [..., K/32] as numbers in 64 bits: sign, exponent and mantissa of e2m1."""
    c = torch.stack((packed % 16, packed // 16), -1).flatten(-2).double()
    sign, rest = 1 - 2 * torch.floor(c / 8), c % 8
    e, m = torch.floor(rest / 2), rest % 2
    v = sign * torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2))
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, group = case["op"], case["group"]
    if op == "quantize":
        return _exact_quantized(_exact_rotate(s["x"].double(), group))
    if op == "linear":
        n, k = case["n"], case["k"]
        x = _exact_quantized(_exact_rotate(s["x"].double(), group))
        r = torch.arange(n, device="cuda")[:, None]
        blk = torch.arange(k // BLOCK, device="cuda")[None, :]
        e = s["wscales"][r // 128, blk // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + blk % 4]
        out = x @ _exact_decoded(s["weight"], e).t()
        return out if s["bias"] is None else out + s["bias"].double()
    if op == "cache":
        page, heads, d = case["page"], case["heads"], case["d"]
        outs = []
        for i, new in enumerate((s["k"], s["v"])):
            held = _exact_decoded(s["codes"][:, i], s["scales"][:, i]).transpose(1, 2).reshape(-1, heads, d)     # by slot
            held[s["write"]] = _exact_quantized(_exact_rotate(new.double(), group))
            outs.append(_exact_rotate(held[s["read"]], group))
        return tuple(outs)
    lens, tq, d, hkv, group_heads = s["lens"].tolist(), case["tq"], case["d"], case["hkv"], case["hq"] // case["hkv"]
    out = torch.zeros(*s["q"].shape, dtype=torch.float64, device="cuda")
    q = _exact_rotate(s["q"].double(), group)
    for b, n in enumerate(lens):
        if not n:
            continue
        pages = s["table"][b, : -(-n // case["page"])].long()
        k, v = (_exact_decoded(s["codes"][pages, i], s["scales"][pages, i]).transpose(0, 1).reshape(hkv, -1, d)[:, :n] for i in (0, 1))
        for t in range(tq):
            sees = n - tq + t + 1
            if sees <= 0:
                continue
            qq = q[b, t].reshape(hkv, group_heads, d)
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", qq, k[:, :sees]) * s["scale"], -1)
            out[b, t] = torch.einsum("hgn,hnd->hgd", p, v[:, :sees]).reshape(-1, d)
    return _exact_rotate(out, group)
