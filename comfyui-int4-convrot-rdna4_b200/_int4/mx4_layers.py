"""Layers on the MX4 operators: a Linear, a paged key/value cache and the
self-attention block that uses both.

``Mx4ConvRotLinear`` holds a weight as MX4 codes (half a byte a value plus one
scale byte per 32) and runs ``convrot_mx4_linear``. ``Mx4KVCache`` owns the
cache's tensors and hands out pages. ``Mx4SelfAttention`` is the path of one
transformer block from hidden states to hidden states: QKV projection, new keys
and values into the cache, attention over it, output projection. Forward only.
"""
from __future__ import annotations

import torch

from . import pick_groupsize
from .mx4 import (
    _scale_tiles,
    convrot_mx4_attention,
    convrot_mx4_cache_append,
    convrot_mx4_cache_read,
    convrot_mx4_linear,
    mx4_cache_empty,
    quantize_convrot_mx4,
)


class Mx4ConvRotLinear(torch.nn.Module):
    """``x @ W.T + bias`` with W held in MX4 (rotated in groups of ``convrot_groupsize``, 0: not rotated).

    State dict: ``weight`` (codes), ``weight_scale`` (tiles), ``bias`` and ``convrot_groupsize``,
    the group that the codes belong to; a dict without the last keeps the module's.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None,
                 convrot_groupsize: int | None = None):
        super().__init__()
        if in_features % 32:
            raise ValueError(f"in_features {in_features} is not a multiple of 32")
        g = convrot_groupsize if convrot_groupsize is not None else (pick_groupsize(in_features) or 0)
        self.in_features, self.out_features, self.groupsize = in_features, out_features, g
        self.register_buffer("weight", torch.zeros(out_features, in_features // 2, dtype=torch.uint8, device=device))
        self.register_buffer("weight_scale", torch.zeros(_scale_tiles(out_features, in_features), dtype=torch.uint8, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=torch.bfloat16, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, convrot_groupsize: int | None = None, device=None) -> "Mx4ConvRotLinear":
        """Quantizes a Linear's weight on a CUDA device (float32, bfloat16 or float16)."""
        device = torch.device(device or linear.weight.device)
        mod = cls(linear.in_features, linear.out_features, linear.bias is not None, device, convrot_groupsize)
        mod.weight, mod.weight_scale = quantize_convrot_mx4(linear.weight.detach().to(device), mod.groupsize)
        if linear.bias is not None:
            mod.bias = linear.bias.detach().to(device)
        return mod

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "convrot_groupsize"] = torch.tensor(self.groupsize)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        key = prefix + "convrot_groupsize"
        if key in state_dict:
            g = int(state_dict[key])
            if g not in (0, 16, 64, 256) or (g and self.in_features % g):
                error_msgs.append(f"{key}: {g} is no rotation group of in_features={self.in_features}")
                return
            self.groupsize = g
        bias = state_dict.get(prefix + "bias")
        if self.bias is not None and bias is not None:
            self.bias = self.bias.to(bias.dtype)                  # (copied into; a checkpoint's type is kept)
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if key in unexpected_keys:
            unexpected_keys.remove(key)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return convrot_mx4_linear(x, self.weight, self.weight_scale, self.bias, self.groupsize)


class Mx4KVCache:
    """The pages of a key/value cache and the sequences that own them.

    ``add`` starts a sequence, ``extend`` reserves the slots of its next tokens (new
    pages are taken when needed; RuntimeError when none is left), ``free`` gives its
    pages back. ``tables`` are what ``convrot_mx4_attention`` takes.
    """

    def __init__(self, pages: int, heads: int, head_dim: int, page: int = 64, convrot_groupsize: int = 64, device="cuda"):
        self.codes, self.scales = mx4_cache_empty(pages, page, heads, head_dim, device)
        self.page, self.groupsize = page, convrot_groupsize
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    def add(self) -> int:
        seq = self._next
        self._next += 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def free(self, seq: int) -> None:
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq]

    def length(self, seq: int) -> int:
        return self._len[seq]

    def extend(self, seq: int, tokens: int) -> list[int]:
        """Slots of the sequence's next ``tokens`` tokens."""
        pages, start = self._pages[seq], self._len[seq]
        need = -(-(start + tokens) // self.page) - len(pages)
        if need > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {need} needed")
        pages.extend(self._free.pop() for _ in range(need))
        self._len[seq] = start + tokens
        return [pages[j // self.page] * self.page + j % self.page for j in range(start, start + tokens)]

    def slots(self, seq: int) -> list[int]:
        """Slots of all of the sequence's tokens."""
        return [self._pages[seq][j // self.page] * self.page + j % self.page for j in range(self._len[seq])]

    def tables(self, seqs) -> tuple[torch.Tensor, torch.Tensor]:
        """(block_table int32 [B, P], seq_lens int32 [B]) of sequences, on the cache's device."""
        width = max(1, max(len(self._pages[s]) for s in seqs))
        rows = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in seqs]
        device = self.codes.device
        return (torch.tensor(rows, dtype=torch.int32, device=device),
                torch.tensor([self._len[s] for s in seqs], dtype=torch.int32, device=device))

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        convrot_mx4_cache_append(self.codes, self.scales, k, v, slots, self.groupsize)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        return convrot_mx4_cache_read(self.codes, self.scales, slots, dtype, self.groupsize)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               softmax_scale: float | None = None) -> torch.Tensor:
        return convrot_mx4_attention(q, self.codes, self.scales, block_table, seq_lens, softmax_scale, self.groupsize)


class Mx4SelfAttention(torch.nn.Module):
    """Causal self-attention of new tokens over a paged MX4 cache, with MX4 projections.

    No position embedding. A model that has one calls the parts itself: ``project``,
    its embedding of q and k, ``cache.append``, ``cache.attend``, ``out``.
    """

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, bias: bool = False, device=None):
        super().__init__()
        if heads % kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {kv_heads} key/value heads")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.qkv = Mx4ConvRotLinear(hidden, (heads + 2 * kv_heads) * head_dim, bias, device)
        self.out = Mx4ConvRotLinear(heads * head_dim, hidden, bias, device)

    def project(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q [..., heads, D], k and v [..., kv_heads, D] of x [..., hidden]: views of one projection."""
        y = self.qkv(x).unflatten(-1, (self.heads + 2 * self.kv_heads, self.head_dim))
        return y.split((self.heads, self.kv_heads, self.kv_heads), dim=-2)

    def forward(self, x: torch.Tensor, cache: Mx4KVCache, slots: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor) -> torch.Tensor:
        """x [B, T, hidden]: the newest T tokens of B sequences, whose slots (int64 [B * T]),
        pages and lengths (the new tokens included) are given. Few tokens a sequence (decoding,
        drafts to verify): every query row is read against the cache as it is stored."""
        b, t, _ = x.shape
        q, k, v = self.project(x)
        cache.append(k.flatten(0, 1), v.flatten(0, 1), slots)
        return self.out(cache.attend(q, block_table, seq_lens).reshape(b, t, self.heads * self.head_dim))

    def prefill(self, x: torch.Tensor, cache: Mx4KVCache, seq: int) -> torch.Tensor:
        """x [T, hidden]: the next T tokens of one sequence. Many query rows: the keys and values
        so far are read back once and torch's attention runs on them."""
        t = x.shape[0]
        device = x.device
        q, k, v = self.project(x)
        new = torch.tensor(cache.extend(seq, t), dtype=torch.int64, device=device)
        cache.append(k, v, new)
        ks, vs = cache.read(torch.tensor(cache.slots(seq), dtype=torch.int64, device=device), x.dtype)
        n = ks.shape[0]
        seen = torch.ones(t, n, dtype=torch.bool, device=device).tril(n - t)
        y = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(0, 1)[None], ks.transpose(0, 1)[None], vs.transpose(0, 1)[None], attn_mask=seen, enable_gqa=True)
        return self.out(y[0].transpose(0, 1).reshape(t, self.heads * self.head_dim))
