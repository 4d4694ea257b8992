"""numpy restatement of the MX4 format and operators (test infrastructure).

``quantize`` rotates in float32 in the kernels' radix-4 order (codes and scales
are then determined bit for bit); ``rotate64``, ``quantize64`` and ``attention64``
are the definitions in 64 bits.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDPOINTS = (GRID[1:] + GRID[:-1]) / 2


def _h4(v, axis):
    v0, v1, v2, v3 = np.moveaxis(v, axis, 0)
    s = (v0 + v1) + (v2 + v3)
    two = v.dtype.type(2)
    return np.stack([s - two * v3, s - two * v2, s - two * v1, s - two * v0], axis=axis)


def rotate(x, group):
    """x [..., K] by the regular Hadamard matrix in groups, in x's own float type:
    radix-4 steps at strides 1, 4, 16, 64, then 1 / sqrt(group)."""
    if not group:
        return x
    digits = {16: 2, 64: 3, 256: 4}[group]
    v = x.reshape(-1, *([4] * digits))
    for axis in range(digits, 0, -1):
        v = _h4(v, axis)
    return (v * x.dtype.type(1 / np.sqrt(group))).reshape(x.shape)


def rotate64(x, group):
    """The same rotation as a matrix product in 64 bits."""
    x = np.asarray(x, np.float64)
    if not group:
        return x
    h4 = np.ones((4, 4)) - 2 * np.fliplr(np.eye(4))
    h = np.ones((1, 1))
    while h.shape[0] < group:
        h = np.kron(h, h4 / 2)
    return (x.reshape(-1, group) @ h).reshape(x.shape)


def encode(x):
    """x [..., K] to codes 0..15 [..., K] and scale bytes [..., K/32]."""
    v = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, BLOCK)
    a = np.abs(v).max(-1)
    bad = ~np.isfinite(a)
    _, e = np.frexp(np.where(bad | (a == 0), 1.0, a))
    e = np.where(a == 0, 0, np.maximum(e - 1 - 2 + 127, 0))
    with np.errstate(invalid="ignore"):
        y = v * np.exp2(127.0 - e)[..., None]
        y = np.where(bad[..., None], 0.0, y)
    m = np.abs(y)
    c = np.searchsorted(MIDPOINTS, m, side="left")            # ties go down ...
    tie = (m[..., None] == MIDPOINTS).any(-1)
    c = np.where(tie & (c % 2 == 1), c + 1, c)                # ... or to the even code
    c = c | (np.signbit(y) << 3)
    return c.reshape(x.shape).astype(np.uint8), np.where(bad, 255, e).astype(np.uint8)


def decode(codes, scales):
    """Codes 0..15 [..., K], scale bytes [..., K/32] -> float64 values."""
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    f = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(f, BLOCK, axis=-1)


def quantize(x32, group):
    return encode(rotate(np.asarray(x32, np.float32), group))


def quantize64(x, group):
    return encode(rotate64(x, group))


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], packed.shape[-1] * 2)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def untile(tiles, rows, k):
    rt, kt, _ = tiles.shape
    return tiles.reshape(rt, kt, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :k // BLOCK]


def attention64(q, k, v, lens, scale):
    """q [B, Tq, Hq, D]; k, v lists of [n_b, Hkv, D]; (out, sum of p |v|, largest scale * sum |q||k|)."""
    b, tq, hq, d = q.shape
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    reach = np.zeros(q.shape[:3])
    for i in range(b):
        for t in range(tq):
            n = min(lens[i], k[i].shape[0]) - tq + t + 1
            if n <= 0:
                continue
            for h in range(hq):
                hk = h // (hq // k[i].shape[1])
                kk, vv = k[i][:n, hk], v[i][:n, hk]
                s = kk @ q[i, t, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, t, h] = p @ vv
                spread[i, t, h] = p @ np.abs(vv)
                reach[i, t, h] = (np.abs(kk) @ np.abs(q[i, t, h])).max() * abs(scale)
    return out, spread, reach


def rounded_apart(got, ref, dtype):
    """Share of the outputs that are not the nearest value of their type ("bf16" or "f16") to ``ref``."""
    import torch
    near = torch.from_numpy(np.ascontiguousarray(ref)).to({"bf16": torch.bfloat16, "f16": torch.float16}[dtype])
    return float((near.double() != torch.from_numpy(np.ascontiguousarray(got, np.float64))).double().mean())


# Operands of attention as the sum of f16 values leave a relative error of at most 2^-22 a
# factor; a score sums up to some 2^5 in magnitude, so weights and outputs are within 2^-17.
# An output is then rounded to another value than the nearest only where it lies that near
# to the middle of two: 2^-17 over the spacing, which is at least 2^-8 (bf16) or 2^-11 (f16)
# of the output. Shares of the outputs:
MOST_APART = {"bf16": 2.0 ** -9, "f16": 2.0 ** -6}


def attention_f16_terms(q, k, v, scale, terms):
    """One head's attention q [R, D], k, v [N, D] with queries and weights as sums of ``terms`` f16 values."""
    def cut(x):
        left, held = x, np.zeros_like(x)
        for _ in range(terms):
            part = left.astype(np.float16).astype(np.float64)
            held, left = held + part, left - part
        return held
    up = np.exp2(8 - np.floor(np.log2(np.abs(q).max(-1, keepdims=True))))
    s = cut(q * up) / up @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    return cut(p) @ v / p.sum(-1, keepdims=True)
