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
"""
from __future__ import annotations

import torch

from .cuda_loader import _check, _IN_DTYPE_CODE, _load

BLOCK = 32
_GROUPS = (0, 16, 64, 256)
_HEAD_DIMS = (64, 128, 256)


def _device_of(*tensors):
    """The one CUDA device of the tensors (None entries skipped); ValueError otherwise."""
    device = None
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                raise ValueError("the B200 ConvRot kernels need CUDA tensors")
            if device is None:
                device = t.device
            elif t.device != device:
                raise ValueError(f"tensors on {device} and {t.device}")
    return device


# the current stream as a number, without building a Stream object for each call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(device, name, *args):
    """Calls a C entry with the device current and its current stream as the last argument."""
    fn = getattr(_load(), name)
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _check(name, rc)


def _group(k: int, group) -> int:
    group = 0 if group is None else group
    if group not in _GROUPS:
        raise ValueError(f"convrot_groupsize must be 16, 64, 256 or 0 (not rotated), got {group!r}")
    if k <= 0 or k % BLOCK:
        raise ValueError(f"MX4 needs a last dimension that is a positive multiple of {BLOCK}, got {k}")
    if group and k % group:
        raise ValueError(f"K={k} not divisible by convrot_groupsize {group}")
    return group


def _dtype_code(dtype) -> int:
    code = _IN_DTYPE_CODE.get(dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}: float32, bfloat16 or float16")
    return code


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as a matrix whose rows are contiguous (a view where strides allow it)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _scale_tiles(rows: int, k: int) -> tuple[int, int, int]:
    return (rows + 127) // 128, (k + 127) // 128, 512


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, what: str) -> tuple[int, int]:
    """(rows, K) of packed codes [..., K/2] and their tiled scales."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"{what} codes and scales must be uint8")
    if codes.dim() < 1 or not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{what} codes and scales must be contiguous")
    k = codes.shape[-1] * 2
    rows = codes.numel() // codes.shape[-1] if k else 0
    if tuple(scales.shape) != _scale_tiles(rows, k):
        raise ValueError(f"{what} scales {tuple(scales.shape)} do not match codes {tuple(codes.shape)}: "
                         f"expected {_scale_tiles(rows, k)}")
    return rows, k


def quantize_convrot_mx4(x: torch.Tensor, convrot_groupsize: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotates the rows of x [..., K] in groups and quantizes them to MX4.

    x float32, bfloat16 or float16, K a multiple of 32 and of the group; a matrix
    may have any row stride. Returns codes uint8 [..., K/2] and scales uint8
    [ceil(R/128), ceil(K/128), 512] for the R rows. Weights are quantized with the
    same call. A block holding an infinity or a NaN stands for NaN as a whole.
    """
    device = _device_of(x)
    if x.dim() < 1:
        raise ValueError("quantize_convrot_mx4 needs at least one dimension")
    k = x.shape[-1]
    group = _group(k, convrot_groupsize)
    code = _dtype_code(x.dtype)
    x2 = _rows(x)
    m = x2.shape[0]
    codes = x2.new_empty((*x.shape[:-1], k // 2), dtype=torch.uint8)
    scales = x2.new_empty(_scale_tiles(m, k), dtype=torch.uint8)
    _call(device, "ck_mx4_quant", x2.data_ptr(), code, x2.stride(0), codes.data_ptr(), scales.data_ptr(), m, k, group)
    return codes, scales


def dequantize_convrot_mx4(codes: torch.Tensor, scales: torch.Tensor, convrot_groupsize: int = 0,
                           dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that MX4 codes [..., K/2] and tiled scales stand for, [..., K] in ``dtype``.

    With a group the rows are rotated back (fp32) before the one rounding to
    ``dtype``; with 0, the default, the values of the rotated rows come back: exact
    in bfloat16 and float32.
    """
    device = _device_of(codes, scales)
    rows, k = _check_codes(codes, scales, "MX4")
    group = _group(k, convrot_groupsize)
    out = codes.new_empty((*codes.shape[:-1], k), dtype=dtype)
    _call(device, "ck_mx4_dequant", codes.data_ptr(), scales.data_ptr(), out.data_ptr(), _dtype_code(dtype), rows, k, group)
    return out


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
    device = _device_of(x, qweight, wscales, bias)
    if qweight.dim() != 2:
        raise ValueError(f"qweight must be [N, K/2], got {tuple(qweight.shape)}")
    n, k = _check_codes(qweight, wscales, "weight")
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"Input K={x.shape[-1] if x.dim() else 0} does not match qweight K={k}")
    group = _group(k, convrot_groupsize)
    code = _dtype_code(x.dtype)
    bias_ptr = bias_code = 0
    if bias is not None:
        if bias.shape != (n,) or bias.dtype not in _IN_DTYPE_CODE:
            raise ValueError(f"bias must be [{n}] in float32, bfloat16 or float16")
        bias = bias.contiguous()
        bias_ptr, bias_code = bias.data_ptr(), _IN_DTYPE_CODE[bias.dtype]
    x2 = _rows(x)
    m = x2.shape[0]
    out = x2.new_empty((*x.shape[:-1], n))
    need = _load().ck_mx4_linear_workspace_size(m, k)
    workspace = x2.new_empty((need,), dtype=torch.uint8) if need else None
    _call(device, "ck_mx4_linear", x2.data_ptr(), code, x2.stride(0), qweight.data_ptr(), wscales.data_ptr(), bias_ptr,
          bias_code, out.data_ptr(), m, n, k, group, workspace.data_ptr() if need else 0, need)
    return out


# --------------------------------------------------------------------- paged cache


def mx4_cache_empty(pages: int, page: int, heads: int, head_dim: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """A zeroed paged cache: codes [pages, 2, heads, page, D/2] and scales [pages, 2, heads, page, D/32]."""
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
    if page <= 0 or page & (page - 1):
        raise ValueError(f"the page size must be a power of two, got {page}")
    codes = torch.zeros(pages, 2, heads, page, head_dim // 2, dtype=torch.uint8, device=device)
    scales = torch.zeros(pages, 2, heads, page, head_dim // BLOCK, dtype=torch.uint8, device=device)
    return codes, scales


def _check_cache(codes, scales, convrot_groupsize):
    """(pages, heads, D, page, group) of a cache."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("cache codes and scales must be uint8")
    if codes.dim() != 5 or codes.shape[1] != 2 or not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("cache codes must be contiguous [pages, 2, heads, page, D/2]")
    pages, _, heads, page, half = codes.shape
    d = 2 * half
    if d not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {d}")
    if scales.shape != (pages, 2, heads, page, d // BLOCK):
        raise ValueError(f"cache scales {tuple(scales.shape)} do not match codes {tuple(codes.shape)}")
    return pages, heads, d, page, _group(d, convrot_groupsize)


def _check_slots(slots, t):
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous() or (t is not None and slots.shape[0] != t):
        raise ValueError("slots must be a contiguous int64 vector, one a token")


def convrot_mx4_cache_append(codes: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             slots: torch.Tensor, convrot_groupsize: int = 64) -> None:
    """Rotates and quantizes new keys and values and writes them to their slots.

    k, v [T, heads, D] (bf16, fp16 or fp32; any token and head strides, D
    contiguous), slots int64 [T]. A slot outside the cache (-1, say) is skipped;
    two tokens of one call must not share a slot.
    """
    device = _device_of(codes, scales, k, v, slots)
    pages, heads, d, page, group = _check_cache(codes, scales, convrot_groupsize)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (heads, d) or k.dtype != v.dtype:
        raise ValueError(f"keys {tuple(k.shape)} and values {tuple(v.shape)} must both be [T, {heads}, {d}] of one dtype")
    t = k.shape[0]
    _check_slots(slots, t)
    code = _dtype_code(k.dtype)
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    _call(device, "ck_mx4_cache_append", codes.data_ptr(), scales.data_ptr(), pages, heads, d, page, group, k.data_ptr(),
          v.data_ptr(), code, k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(), t)


def convrot_mx4_cache_read(codes: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor,
                           dtype: torch.dtype = torch.bfloat16, convrot_groupsize: int = 64
                           ) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [T, heads, D] held at ``slots`` (int64 [T]), rotated back, in ``dtype``;
    a slot outside the cache reads as zeros."""
    device = _device_of(codes, scales, slots)
    pages, heads, d, page, group = _check_cache(codes, scales, convrot_groupsize)
    _check_slots(slots, None)
    t = slots.shape[0]
    code = _dtype_code(dtype)
    k = codes.new_empty((t, heads, d), dtype=dtype)
    v = codes.new_empty((t, heads, d), dtype=dtype)
    _call(device, "ck_mx4_cache_read", codes.data_ptr(), scales.data_ptr(), pages, heads, d, page, group, slots.data_ptr(),
          t, k.data_ptr(), v.data_ptr(), code)
    return k, v


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
    gives zeros. Returns [B, Tq, Hq, D] in q.dtype.
    """
    device = _device_of(q, codes, scales, block_table, seq_lens)
    pages, heads, d, page, group = _check_cache(codes, scales, convrot_groupsize)
    if q.dim() != 4 or q.shape[3] != d or q.shape[1] == 0 or q.shape[2] == 0 or q.shape[2] % heads:
        raise ValueError(f"q {tuple(q.shape)} must be [B, Tq, a multiple of {heads}, {d}]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"queries must be bfloat16 or float16, got {q.dtype}")
    b, tq, hq, _ = q.shape
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != b or \
            (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("block_table must be int32 [B, pages of a sequence] with contiguous rows")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (b,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 vector [B]")
    if q.stride(3) != 1:
        q = q.contiguous()
    per_seq = block_table.shape[1]
    out = q.new_empty((b, tq, hq, d))
    need = _load().ck_mx4_attention_workspace_size(b, tq, hq, heads, d, per_seq * page)
    workspace = q.new_empty((need,), dtype=torch.uint8) if need else None
    _call(device, "ck_mx4_attention", q.data_ptr(), _IN_DTYPE_CODE[q.dtype], q.stride(0), q.stride(1), q.stride(2),
          codes.data_ptr(), scales.data_ptr(), pages, page, block_table.data_ptr(), max(block_table.stride(0), per_seq),
          per_seq, seq_lens.data_ptr(), out.data_ptr(), b, tq, hq, heads, d, group,
          d ** -0.5 if softmax_scale is None else float(softmax_scale), workspace.data_ptr() if need else 0, need)
    return out
