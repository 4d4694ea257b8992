"""Microscaled 4-bit floats (MX4: OCP MXFP4) with the ConvRot rotation.

The format next to the package's int4: 4-bit floats e2m1 in blocks of 32, each
block with one power-of-two scale byte (E8M0), a form the B200 tensor cores
multiply as it is stored. Rows are rotated by the same regular Hadamard matrix
as the int4 path (groups of 16, 64 or 256; 0: not rotated) in fp32, without an
intermediate rounding.

    quantize_convrot_mx4(x, G) -> (codes, scales)
    dequantize_convrot_mx4(codes, scales, G, dtype) -> values
    convrot_mx4_linear(x, qweight, wscales, bias, G) -> x @ W.T + bias
    convrot_mx4_cache_append(codes, scales, k, v, slots, G)
    convrot_mx4_cache_read(codes, scales, slots, dtype, G) -> (k, v)
    convrot_mx4_attention(q, codes, scales, block_table, seq_lens, ...) -> out

Layouts. Codes: two a byte, the even column in the low nibble. Scales of a
matrix [R, K] are held in tiles [ceil(R/128), ceil(K/128), 512] (the order in
which the tensor cores take them): the byte of row r and block b sits at
(r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 of tile (r / 128, b / 4);
``mx4_scales_to_rows`` / ``mx4_scales_from_rows`` convert to and from [R, K/32].
A cache is codes [pages, 2, heads, page, D/2] and scales [pages, 2, heads, page,
D/32] (``mx4_cache_empty``), keys at index 0 and values at 1, both rotated along
D; slot s is token s % page of page s / page.

All tensors are CUDA tensors of one device; calls run on that device's current
stream; bad arguments raise ValueError, a refused or failed launch RuntimeError.
Forward only, like the int4 operators: no result carries a gradient, whether the
inputs require one or not.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os
import threading

import torch

from . import build as _build
from . import cuda_loader

BLOCK = 32
_HEAD_DIMS = (64, 128, 256)

_native = None
_lock = threading.Lock()


def native():
    """The binding module (built first when there is none for these sources and this torch)."""
    global _native
    if _native is None:
        with _lock:
            if _native is None:
                cuda_loader.library()
                path = _build.binding_path()
                if not os.path.exists(path):
                    _build.build_binding()
                loader = importlib.machinery.ExtensionFileLoader("_mx4_binding", path)
                spec = importlib.util.spec_from_loader("_mx4_binding", loader)
                module = importlib.util.module_from_spec(spec)
                loader.exec_module(module)
                _native = module
    return _native


def _scale_tiles(rows: int, k: int) -> tuple[int, int, int]:
    return (rows + 127) // 128, (k + 127) // 128, 512


def quantize_convrot_mx4(x: torch.Tensor, convrot_groupsize: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotates the rows of x [..., K] in groups and quantizes them to MX4.

    x float32, bfloat16 or float16, K a multiple of 32 and of the group; a matrix
    may have any row stride. Returns codes uint8 [..., K/2] and scales uint8
    [ceil(R/128), ceil(K/128), 512] for the R rows. Weights are quantized with the
    same call. A block holding an infinity or a NaN stands for NaN as a whole.
    """
    return (_native or native()).quantize(x, convrot_groupsize)


def dequantize_convrot_mx4(codes: torch.Tensor, scales: torch.Tensor, convrot_groupsize: int = 0,
                           dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that MX4 codes [..., K/2] and tiled scales stand for, [..., K] in ``dtype``.

    With a group the rows are rotated back (fp32) before the one rounding to
    ``dtype``; with 0, the default, the values of the rotated rows come back: exact
    in bfloat16 and float32.
    """
    return (_native or native()).dequantize(codes, scales, convrot_groupsize, dtype)


def mx4_scales_to_rows(scales: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """Tiled scales as a row-major matrix [rows, K/32] (any device)."""
    if tuple(scales.shape) != _scale_tiles(rows, k) or k % BLOCK:
        raise ValueError(f"scales {tuple(scales.shape)} are not the tiles of a {rows} x {k} matrix")
    rt, kt, _ = scales.shape
    full = scales.reshape(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)
    return full[:rows, :k // BLOCK].contiguous()


def mx4_scales_from_rows(scales: torch.Tensor) -> torch.Tensor:
    """Row-major scale bytes [R, K/32] (as MXFP4 checkpoints hold them) in tiles (any device)."""
    if scales.dim() != 2 or scales.dtype != torch.uint8:
        raise ValueError("expected uint8 scales [R, K/32]")
    r, b = scales.shape
    rt, kt = (r + 127) // 128, (b + 3) // 4
    full = scales.new_zeros(rt * 128, kt * 4)
    full[:r, :b] = scales
    return full.reshape(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512).contiguous()


def convrot_mx4_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor, bias: torch.Tensor | None = None,
                       convrot_groupsize: int = 256) -> torch.Tensor:
    """``x @ W.T + bias`` with x quantized to MX4 on the way and W held in MX4.

    x [..., K] (bf16, fp16 or fp32), qweight uint8 [N, K/2] and wscales from
    ``quantize_convrot_mx4(W, convrot_groupsize)`` with the same group, bias [N] in
    any of the three dtypes or None. fp32 accumulation, one rounding; returns
    [..., N] in x.dtype.
    """
    return (_native or native()).linear(x, qweight, wscales, bias, convrot_groupsize)


# --------------------------------------------------------------------- paged cache


def mx4_cache_empty(pages: int, page: int, heads: int, head_dim: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """A zeroed paged cache: codes [pages, 2, heads, page, D/2] and scales [pages, 2, heads, page, D/32]."""
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
    if page <= 0 or page & (page - 1) or page > 65536:
        raise ValueError(f"the page size must be a power of two up to 65536, got {page}")
    if heads <= 0:
        raise ValueError("the cache has no heads")
    codes = torch.zeros(pages, 2, heads, page, head_dim // 2, dtype=torch.uint8, device=device)
    scales = torch.zeros(pages, 2, heads, page, head_dim // BLOCK, dtype=torch.uint8, device=device)
    return codes, scales


def convrot_mx4_cache_append(codes: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             slots: torch.Tensor, convrot_groupsize: int = 64) -> None:
    """Rotates and quantizes new keys and values and writes them to their slots.

    k, v [T, heads, D] (bf16, fp16 or fp32; any token and head strides, D
    contiguous), slots int64 [T]. A slot outside the cache (-1, say) is skipped;
    two tokens of one call must not share a slot.
    """
    (_native or native()).cache_append(codes, scales, k, v, slots, convrot_groupsize)


def convrot_mx4_cache_read(codes: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor,
                           dtype: torch.dtype = torch.bfloat16, convrot_groupsize: int = 64
                           ) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [T, heads, D] held at ``slots`` (int64 [T]), rotated back, in ``dtype``;
    a slot outside the cache reads as zeros."""
    return (_native or native()).cache_read(codes, scales, slots, dtype, convrot_groupsize)


def convrot_mx4_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                          seq_lens: torch.Tensor, softmax_scale: float | None = None,
                          convrot_groupsize: int = 64) -> torch.Tensor:
    """Causal attention of each sequence's newest tokens over the paged cache.

    q [B, Tq, Hq, D] (bf16 or fp16; any strides but a contiguous D): the queries of
    the last Tq tokens, whose keys and values are in the cache already. Hq is a
    multiple of the cache's heads (query head h reads cache head h * heads / Hq).
    block_table int32 [B, P]: token j of sequence b is token j % page of page
    block_table[b, j / page]; a page number outside the cache hides its tokens.
    seq_lens int32 [B]: tokens in the cache, new ones included (cut at P * page).
    Query t sees the tokens up to position seq_len - Tq + t; a query that sees none
    gives zeros. Returns [B, Tq, Hq, D] in q.dtype. Keys of a magnitude beyond 2^111
    may overflow the scores' partial sums.
    """
    return (_native or native()).attention(q, codes, scales, block_table, seq_lens, softmax_scale, convrot_groupsize)
