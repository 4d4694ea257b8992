"""The operators of a transformer block around the MX4 cache: what is timed and compared.

Four operators, in the order in which a block that verifies drafted tokens runs them:

* ``norm``: a residual is added, the rows are divided by their root mean square, rotated,
  quantized to 8 bits with a scale a row and multiplied by a weight held in 8 bits (W8A8).
* ``rope``: queries and keys are turned by their tokens' positions, which have one axis (text)
  or several (image: index, height, width).
* ``append``: the same for the queries, keys and values of new tokens on the way into a paged
  MX4 cache (4-bit floats in blocks of 32 with a power-of-two scale, rotated by a Hadamard
  matrix); the keys and values are then read back, as the chunk's own attention does.
* ``tree``: attention of a tree of drafted tokens over the paged MX4 cache: each node sees the
  sequence so far and the nodes that its row of the mask names (its ancestors and itself).

Definitions.
norm: h = x + r; y = R(h / sqrt(mean h^2 + eps) * g); s = max(max |y|, 1e-10) / 127; c = round(y / s),
  ties to even; out = (c . w) s s_w + bias; h is returned too. R: the regular Hadamard matrix in groups.
rope: pair i of a head, channels (2i, 2i + 1) or (i, i + P), is turned by the angle p_a f_i, a the
  axis to whose section i belongs; the channels behind the 2P first stay as they are.
tree: out = sum_j exp(s_tj) v_j / sum_j exp(s_tj), s_tj = scale q_t k_j, over the tokens j that node t
  sees; zeros where there are none, and for the padding behind a sequence's nodes.

Cache: codes [pages, 2, heads, page, D/2] and scales [pages, 2, heads, page, D/32], keys at index 0
and values at 1, both rotated along D, two codes a byte, the even column in the low nibble.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
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
        # one decoded token ahead of the MLP's up projection: the weight's bytes
        {"name": "norm_one_token", "op": "norm", "m": 1, "n": 15360, "k": 3840, "group": 256, "residual": True, "bias": False, "dtype": "bf16"},
        # a short prompt (odd count) ahead of a query, key and value projection, with bias
        {"name": "norm_text", "op": "norm", "m": 509, "n": 6144, "k": 4096, "group": 64, "residual": True, "bias": True, "dtype": "bf16"},
        # image tokens of the largest size of the token sweep, the first block (no residual yet)
        {"name": "norm_image", "op": "norm", "m": 16384, "n": 15360, "k": 3840, "group": 256, "residual": False, "bias": True, "dtype": "bf16"},
        # one decoded token far into a conversation: latency only
        {"name": "rope_one_token", "op": "rope", "b": 1, "t": 1, "h": 40, "d": 128, "sections": "64", "far": 100000, "floats": False,
         "interleaved": False, "inverse": False, "order": "bthd", "dtype": "bf16"},
        # the rotation back (a gradient, keys that move), half of the channels, an odd count of tokens of two prompts, heads outside
        {"name": "rope_back", "op": "rope", "b": 2, "t": 509, "h": 24, "d": 64, "sections": "16", "far": 2048, "floats": False,
         "interleaved": False, "inverse": True, "order": "bhtd", "dtype": "f16"},
        # queries and keys of a 1024 x 1024 image and its text, three axes
        {"name": "rope_image", "op": "rope", "b": 1, "t": 4608, "h": 60, "d": 128, "sections": "8,28,28", "far": 64, "floats": True,
         "interleaved": True, "inverse": False, "order": "bthd", "dtype": "bf16"},
        # one decode step of a small batch
        {"name": "append_decode", "op": "append", "new": 7, "hq": 32, "hkv": 8, "d": 128, "page": 16, "group": 64, "sections": "64", "far": 30000,
         "interleaved": False, "dtype": "bf16"},
        # a chunk of a prompt with images in it: three axes, an odd count of tokens
        {"name": "append_chunk", "op": "append", "new": 2047, "hq": 24, "hkv": 8, "d": 64, "page": 32, "group": 16, "sections": "8,12,12", "far": 4096,
         "interleaved": False, "dtype": "f16"},
        # several long prompts at once
        {"name": "append_prompts", "op": "append", "new": 32768, "hq": 32, "hkv": 8, "d": 128, "page": 64, "group": 64, "sections": "64", "far": 32768,
         "interleaved": False, "dtype": "bf16"},
        # one user's short conversation, a small tree
        {"name": "tree_short", "op": "tree", "b": 1, "t": 8, "hq": 32, "hkv": 8, "d": 128, "page": 64, "group": 64, "longest": 777,
         "ragged": False, "dtype": "bf16"},
        # a ragged batch with empty slots, trees of different sizes
        {"name": "tree_batch", "op": "tree", "b": 37, "t": 24, "hq": 24, "hkv": 8, "d": 64, "page": 16, "group": 64, "longest": 4096,
         "ragged": True, "dtype": "f16"},
        # long contexts, a wide tree each
        {"name": "tree_long", "op": "tree", "b": 8, "t": 64, "hq": 64, "hkv": 8, "d": 128, "page": 64, "group": 64, "longest": 16384,
         "ragged": False, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def _sections(rng, d):
    """Pairs of each axis: all of the head's or half of them, on one axis, two or three."""
    pairs = d // 2 if rng.random() < 0.7 else d // 4
    axes = rng.choice((1, 1, 2, 3))
    if axes == 1:
        return str(pairs)
    first = max(1, pairs // 8)
    if axes == 2:
        return "%d,%d" % (first, pairs - first)
    rest = (pairs - first) // 2
    return "%d,%d,%d" % (first, rest, pairs - first - rest)


def draw(rng):
    op = rng.choice(("norm", "rope", "append", "tree"))
    if op == "norm":
        group = rng.choice((16, 64, 256))
        k = group * _between(rng, max(1, 512 // group), 15360 // group)
        m = _between(rng, 1, 16384)
        n = _between(rng, 64, min(15360, 16384 * 15360 * 3840 // (m * k)))
        return {"op": op, "m": m, "n": n, "k": k, "group": group, "residual": rng.random() < 0.7, "bias": rng.random() < 0.5,
                "dtype": rng.choice(("bf16", "f16"))}
    d = rng.choice((64, 128, 256))
    if op == "rope":
        h, b = _between(rng, 1, 64), rng.choice((1, 1, 2, 5))
        t = _between(rng, 1, min(16384, 4608 * 60 * 128 // (h * d * b)))
        return {"op": op, "b": b, "t": t, "h": h, "d": d, "sections": _sections(rng, d), "far": _between(rng, 16, 1000000),
                "floats": rng.random() < 0.4, "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3,
                "order": rng.choice(("bthd", "bhtd")), "dtype": rng.choice(("bf16", "f16", "f32"))}
    group = rng.choice((0, 16, 64))
    page = rng.choice((16, 32, 64, 128))
    hkv = rng.choice((1, 2, 4, 8, 16))
    hq = hkv * rng.choice((1, 2, 3, 4, 8))
    if op == "append":
        new = _between(rng, 1, min(32768, 32768 * 48 * 128 // ((hq + 2 * hkv) * d)))
        return {"op": op, "new": new, "hq": hq, "hkv": hkv, "d": d, "page": page, "group": rng.choice((16, 64)), "sections": _sections(rng, d),
                "far": _between(rng, 16, 1000000), "interleaved": rng.random() < 0.4, "dtype": rng.choice(("bf16", "f16"))}
    b, t = _between(rng, 1, 64), _between(rng, 1, 256)
    most = 8 * 64 * 64 * 16384 * 128 // (b * t * hq * d)
    longest = _between(rng, 1, max(1, min(131072, most, 8 * 16384 * 8 * 128 * 16 // (b * hkv * d))))
    return {"op": op, "b": b, "t": t, "hq": hq, "hkv": hkv, "d": d, "page": page, "group": group, "longest": max(longest, t),
            "ragged": rng.random() < 0.7, "dtype": rng.choice(("bf16", "f16"))}


def work(case):
    op = case["op"]
    if op == "norm":
        m, n, k, size = case["m"], case["n"], case["k"], DTYPES[case["dtype"]].itemsize
        return {"bytes": m * k * size * (3 if case["residual"] else 1) + n * k + 4 * n + m * n * size + (size * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    axes = len(case["sections"].split(",")) if op != "tree" else 0
    if op == "rope":
        n = case["b"] * case["t"] * case["h"] * case["d"]
        return {"bytes": 2 * n * DTYPES[case["dtype"]].itemsize + case["b"] * case["t"] * axes * (4 if case["floats"] else 8), "flops": 3 * n}
    if op == "append":
        q, kv = case["hq"] * case["d"], 2 * case["hkv"] * case["d"]
        return {"bytes": case["new"] * (4 * q + kv * (2 + 17 / 32) + 8 + 8 * axes + kv * (2 + 17 / 32) + 8), "flops": 3 * case["new"] * (q + kv)}
    # the lengths of a ragged batch go by the seed: half the longest on average
    b, t = case["b"], case["t"]
    tokens = b * case["longest"] if not case["ragged"] else case["longest"] * (1 + max(0, b - 1) / 2)
    rows = t * case["hq"]
    return {"bytes": tokens * case["hkv"] * case["d"] * 2 * 17 / 32 + 2 * 2 * b * rows * case["d"] + b * t * t, "flops": 4 * tokens * rows * case["d"]}


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
        v = _h4(_h4(x.reshape(-1, 4, 4), 2), 1)
    elif group == 64:
        v = _h4(_h4(_h4(x.reshape(-1, 4, 4, 4), 3), 2), 1)
    else:
        v = _h4(_h4(_h4(_h4(x.reshape(-1, 4, 4, 4, 4), 4), 3), 2), 1)
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


def _plain_norm(s):
    x = s["x"]
    h = x.float() if s["r"] is None else x.float() + s["r"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["g"].float()
    y = _rotate(y, s["group"])
    scale = y.abs().amax(-1, keepdim=True).clamp_min(1e-10) / 127
    c = torch.round(y / scale).clamp(-127, 127)
    out = (c @ s["w"].float().t()) * scale * s["ws"]
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(x.dtype), h.to(x.dtype)


def _turned(x, positions, freqs, sections, interleaved, inverse=False):
    """x [..., T, H, D] turned, in 32 bits; the angles in 64. positions [..., T] or [..., T, axes]."""
    p = positions.double().reshape(*x.shape[:-2], len(sections))
    p = torch.cat([p[..., i:i + 1].expand(*p.shape[:-1], n) for i, n in enumerate(sections)], -1)
    angle = (p * freqs).unsqueeze(-2)
    c, s = angle.cos().float(), angle.sin().float()
    if inverse:
        s = -s
    n, x = freqs.numel(), x.float()
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def _plain_rope(s):
    return _turned(s["x"], s["positions"], s["freqs"], s["sections"], s["interleaved"], s["inverse"]).to(s["x"].dtype)


def _plain_append(s):
    page = s["codes"].shape[3]
    at, off = s["slots"] // page, s["slots"] % page
    how = (s["positions"], s["freqs"], s["sections"], s["interleaved"])
    held = []
    for i, new in enumerate((_turned(s["k"], *how), s["v"].float())):
        c, e = _encode(_rotate(new, s["group"]))
        s["codes"][at, i, :, off] = _pack(c)
        s["scales"][at, i, :, off] = e
        held.append(_rotate(_values(_unpack(s["codes"][at, i, :, off]), s["scales"][at, i, :, off]), s["group"]).to(s["k"].dtype))
    return _turned(s["q"], *how).to(s["q"].dtype), *held


def _plain_tree(s):
    q, table, lens, nodes = s["q"], s["table"].long(), s["lens"].long(), s["nodes"].long()
    b, t, hq, d = q.shape
    _, _, hkv, page, _ = s["codes"].shape
    n = table.shape[1] * page
    qr = _rotate(q.float(), s["group"]).reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4)      # [b, heads, t, group, d]

    def gathered(i):
        c, e = s["codes"][table, i], s["scales"][table, i]                       # [b, pages, heads, page, .]
        return _values(_unpack(c), e).transpose(1, 2).reshape(b, hkv, n, d)

    node = torch.arange(n, device=q.device) - (lens - nodes)[:, None]            # [b, n] a token's number among the nodes, negative: context
    named = torch.gather(s["mask"].expand(b, t, t), 2, node.clamp(0, t - 1)[:, None].expand(b, t, n))
    seen = (node < 0)[:, None] | (named & (node < nodes[:, None])[:, None])      # [b, t, n]
    seen = seen & (torch.arange(t, device=q.device) < nodes[:, None])[..., None]
    score = (qr.reshape(b, hkv, -1, d) @ gathered(0).transpose(2, 3)).reshape(b, hkv, t, hq // hkv, n) * s["scale"]
    score = torch.where(seen[:, None, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = _rotate((p.reshape(b, hkv, -1, n) @ gathered(1)).reshape(b, hkv, t, hq // hkv, d), s["group"])
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)


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


def _axes(case):
    return tuple(int(n) for n in case["sections"].split(","))


def _freqs(sections, theta=10000.0):
    """The usual frequencies theta^(-i / n) of each axis's n pairs, in 64 bits."""
    return torch.cat([theta ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections]).cuda()


def _positions(shape, case, g, dtype):
    """Whole numbers up to the farthest; one axis: tokens in a row."""
    far, axes = case["far"], len(_axes(case))
    if axes > 1:
        return torch.randint(0, far + 1, (*shape, axes), generator=g, device="cuda").to(dtype)
    start = torch.randint(0, far + 1, (*shape[:-1], 1), generator=g, device="cuda")
    return (start + torch.arange(shape[-1], device="cuda")).to(dtype)


def _trees(case, seed):
    """Lengths, nodes and mask [b, t, t] of a batch: host data that a scheduler has. A node's parent is a node before it, or the
    sequence's last token. Ragged batches hold an empty slot, a sequence of its nodes alone and the longest."""
    b, t, longest = case["b"], case["t"], case["longest"]
    rng = random.Random(1000003 * seed + b)
    lens, nodes = [longest] * b, [t] * b
    if case["ragged"]:
        nodes = [t if i == 0 else 0 if i == 1 else rng.randint(1, t) for i in range(b)]
        lens = [longest if i == 0 else 0 if i == 1 else nodes[i] if i == 2 else rng.randint(nodes[i], longest) for i in range(b)]
    of = torch.Generator().manual_seed(seed)
    parents = (torch.rand(b, t, generator=of) * (torch.arange(t) + 1)).long().clamp(max=torch.arange(t)) - 1
    mask = torch.eye(t, dtype=torch.bool).repeat(b, 1, 1)
    for j in range(1, t):
        p = parents[:, j]
        mask[:, j] |= mask[torch.arange(b), p.clamp(min=0)] & (p >= 0)[:, None]
    return lens, nodes, mask


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "norm":
        m, n, k, group, dtype = (case[x] for x in ("m", "n", "k", "group", "dtype"))
        w = _rotate(torch.randn(n, k, generator=g, device="cuda") * 0.02, group)
        ws = w.abs().amax(-1) / 127
        return {"op": op, "group": group, "x": _activations(m, k, dtype, g), "r": _activations(m, k, dtype, g) if case["residual"] else None,
                "g": (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(DTYPES[dtype]), "w": torch.round(w / ws[:, None]).to(torch.int8), "ws": ws,
                "bias": (torch.randn(n, generator=g, device="cuda") * 0.01).to(DTYPES[dtype]) if case["bias"] else None}
    if op == "rope":
        b, t, h, d = (case[x] for x in ("b", "t", "h", "d"))
        x = torch.randn(*((b, t, h, d) if case["order"] == "bthd" else (b, h, t, d)), generator=g, device="cuda").to(DTYPES[case["dtype"]])
        return {"op": op, "x": x if case["order"] == "bthd" else x.transpose(1, 2), "positions": _positions((b, t), case, g, torch.float32 if case["floats"] else torch.int64),
                "freqs": _freqs(_axes(case)), "sections": _axes(case), "interleaved": case["interleaved"], "inverse": case["inverse"]}
    d, page, group, hq, hkv = (case[x] for x in ("d", "page", "group", "hq", "hkv"))
    if op == "append":
        new = case["new"]
        pages = -(-new // page) + 2
        codes, scales = _cache(pages, hkv, page, d, group, g)
        slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        q, k, v = _activations(new, (hq + 2 * hkv) * d, case["dtype"], g).reshape(new, -1, d).split((hq, hkv, hkv), 1)
        return {"op": op, "group": group, "codes": codes, "scales": scales, "q": q, "k": k, "v": v, "slots": slots.reshape(-1)[:new].contiguous(),
                "positions": _positions((new,), case, g, torch.int64), "freqs": _freqs(_axes(case)), "sections": _axes(case), "interleaved": case["interleaved"]}
    b, t = case["b"], case["t"]
    lens, nodes, mask = _trees(case, seed)
    each = max(1, -(-case["longest"] // page))
    codes, scales = _cache(b * each, hkv, page, d, group, g)
    table = torch.randperm(b * each, generator=g, device="cuda").reshape(b, each).int()
    q = _activations(b * t, hq * d, case["dtype"], g).reshape(b, t, hq, d)
    q = (q.float().clamp(-4, 4)).to(q.dtype)                                      # queries are normalised ahead of attention
    return {"op": op, "group": group, "codes": codes, "scales": scales, "q": q, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "nodes": torch.tensor(nodes, dtype=torch.int32, device="cuda"), "mask": mask.cuda(), "scale": 1 / math.sqrt(d)}


def run(state):
    op, s = state["op"], state
    if not own:
        return {"norm": _plain_norm, "rope": _plain_rope, "append": _plain_append, "tree": _plain_tree}[op](s)
    lib = _package()
    if op == "norm":
        return lib.convrot_w8a8_linear_rmsnorm(s["x"], s["w"], s["ws"], s["bias"], norm_weight=s["g"], residual=s["r"], eps=EPS, convrot_groupsize=s["group"])
    if op == "rope":
        return lib.apply_rope(s["x"], s["positions"], s["freqs"], sections=s["sections"], interleaved=s["interleaved"], inverse=s["inverse"])
    if op == "append":
        q = lib.convrot_mx4_cache_append_rope(s["codes"], s["scales"], s["q"], s["k"], s["v"], s["slots"], s["positions"], s["freqs"],
                                              sections=s["sections"], interleaved=s["interleaved"], convrot_groupsize=s["group"])
        return q, *lib.convrot_mx4_cache_read(s["codes"], s["scales"], s["slots"], dtype=s["k"].dtype, convrot_groupsize=s["group"])
    return lib.convrot_mx4_tree_attention(s["q"], s["codes"], s["scales"], s["table"], s["lens"], s["mask"], tree_lens=s["nodes"],
                                          softmax_scale=s["scale"], convrot_groupsize=s["group"])


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
    """The nearest values of the 4-bit format to x [..., K] (64 bits), ties to the even one."""
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


def _exact_turned(x, s):
    """Pairs as complex numbers times e^(i angle), pair by pair of each axis."""
    out, at = x.double().clone(), 0
    positions = s["positions"].double().reshape(*x.shape[:-2], len(s["sections"]))
    total = sum(s["sections"])
    for axis, n in enumerate(s["sections"]):
        pairs = torch.arange(at, at + n, device=x.device)
        re, im = (2 * pairs, 2 * pairs + 1) if s["interleaved"] else (pairs, pairs + total)
        angle = positions[..., axis, None, None] * s["freqs"][at:at + n]
        z = torch.complex(out[..., re], out[..., im]) * torch.polar(torch.ones_like(angle), -angle if s.get("inverse") else angle)
        out[..., re], out[..., im] = z.real, z.imag
        at += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double() + (0 if s["r"] is None else s["r"].double())
        y = _exact_rotate(h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["k"] + EPS) * s["g"].double(), case["group"])
        top = y.abs().max(-1, keepdim=True).values
        out = (torch.round(y * (127 / top)) @ s["w"].double().t()) * (top / 127) * s["ws"].double()
        return out if s["bias"] is None else out + s["bias"].double(), h
    if op == "rope":
        return _exact_turned(s["x"], s)
    group, page, d, hkv = case["group"], case["page"], case["d"], case["hkv"]
    if op == "append":
        held = (_exact_rotate(_exact_quantized(_exact_rotate(x, group)), group) for x in (_exact_turned(s["k"], s), s["v"].double()))
        return _exact_turned(s["q"], s), *held
    lens, nodes, t, each = s["lens"].tolist(), s["nodes"].tolist(), case["t"], case["hq"] // hkv
    out = torch.zeros(*s["q"].shape, dtype=torch.float64, device="cuda")
    q = _exact_rotate(s["q"].double(), group)
    for b, (n, m) in enumerate(zip(lens, nodes)):
        if not m:
            continue
        pages = s["table"][b, : -(-n // page)].long()
        hidden = torch.zeros(m, 1, n, dtype=torch.bool, device="cuda")
        hidden[:, 0, n - m:] = ~s["mask"][b, :m, :m]
        for head in range(hkv):
            k, v = (_exact_decoded(s["codes"][pages, i, head], s["scales"][pages, i, head]).reshape(-1, d)[:n] for i in (0, 1))
            at = slice(head * each, (head + 1) * each)
            score = torch.einsum("tgd,nd->tgn", q[b, :m, at], k) * s["scale"]
            out[b, :m, at] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return _exact_rotate(out, group)
