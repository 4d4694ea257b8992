"""Layers on the MX4 operators: a Linear, a paged key/value cache and the
self-attention block that uses both.

``Mx4ConvRotLinear`` holds a weight as MX4 codes (half a byte a value plus one
scale byte per 32) and runs ``convrot_mx4_linear``. ``Mx4KVCache`` owns the
cache's tensors and hands out pages. ``Mx4SelfAttention`` is the path of one
transformer block from hidden states to hidden states: QKV projection, positions, new
keys and values into the cache, attention over it (of a chain of tokens or of a tree of
drafted ones), output projection. Forward only.
"""
from __future__ import annotations

import math

import torch

from . import pick_groupsize
from .mx4 import (
    _scale_tiles,
    convrot_mx4_attention,
    convrot_mx4_cache_append,
    convrot_mx4_cache_append_rope,
    convrot_mx4_cache_read,
    convrot_mx4_linear,
    convrot_mx4_tree_attention,
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

    def append_rope(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                    freqs: torch.Tensor, sections: tuple[int, ...] | None = None, interleaved: bool = False) -> torch.Tensor | None:
        return convrot_mx4_cache_append_rope(self.codes, self.scales, q, k, v, slots, positions, freqs, sections, interleaved, self.groupsize)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        return convrot_mx4_cache_read(self.codes, self.scales, slots, dtype, self.groupsize)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               softmax_scale: float | None = None) -> torch.Tensor:
        return convrot_mx4_attention(q, self.codes, self.scales, block_table, seq_lens, softmax_scale, self.groupsize)

    def attend_tree(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, tree_mask: torch.Tensor,
                    tree_lens: torch.Tensor | None = None, softmax_scale: float | None = None) -> torch.Tensor:
        return convrot_mx4_tree_attention(q, self.codes, self.scales, block_table, seq_lens, tree_mask, tree_lens, softmax_scale, self.groupsize)

    def accept(self, seq: int, nodes: int, kept) -> None:
        """Ends a tree's verification: of the sequence's ``nodes`` newest tokens those numbered
        ``kept`` stay (in rising order, a path from the root), the others' tokens and the pages
        behind the last are given back. Keys carry their positions already: a node's depth must
        be its place on the path. Worked out on the host, one sequence a call, four indexing kernels
        where a token moves; it cannot be captured into a graph."""
        kept = [int(i) for i in kept]
        start = self._len[seq] - nodes
        if nodes < 0 or start < 0 or any(not 0 <= i < nodes for i in kept) or any(b <= a for a, b in zip(kept, kept[1:])):
            raise ValueError(f"kept nodes {kept} of the newest {nodes} of {self._len[seq]} tokens")
        slots = self.slots(seq)
        moved = [(slots[start + i], slots[start + to]) for to, i in enumerate(kept) if i != to]
        if moved:
            with torch.inference_mode(self.codes.is_inference()):  # (a cache made there can be written there alone)
                src, dst = torch.tensor(moved, dtype=torch.int64, device=self.codes.device).unbind(1)
                for t in (self.codes, self.scales):               # (read as a whole before it is written)
                    t[dst // self.page, :, :, dst % self.page] = t[src // self.page, :, :, src % self.page]
        self._len[seq] = start + len(kept)
        pages = self._pages[seq]
        while len(pages) > -(-self._len[seq] // self.page):
            self._free.append(pages.pop())


class Mx4SelfAttention(torch.nn.Module):
    """Causal self-attention of new tokens over a paged MX4 cache, with MX4 projections.

    freqs (float64 [pairs], ``rope_freqs``): rotary positions for queries and keys, with
    sections and interleaved as in ``apply_rope`` (there neighbours are the default, here halves); None:
    no position embedding. A model that
    has another one calls the parts itself: ``project``, its embedding of q and k,
    ``cache.append``, ``cache.attend``, ``out``.
    """

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, bias: bool = False, device=None,
                 freqs: torch.Tensor | None = None, sections: tuple[int, ...] | None = None, interleaved: bool = False):
        super().__init__()
        if heads % kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {kv_heads} key/value heads")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.sections, self.interleaved = sections, interleaved
        self.qkv = Mx4ConvRotLinear(hidden, (heads + 2 * kv_heads) * head_dim, bias, device)
        self.out = Mx4ConvRotLinear(heads * head_dim, hidden, bias, device)
        self.register_buffer("freqs", None if freqs is None else freqs.to(device), persistent=False)

    def project(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """q [..., heads, D], k and v [..., kv_heads, D] of x [..., hidden]: views of one projection."""
        y = self.qkv(x).unflatten(-1, (self.heads + 2 * self.kv_heads, self.head_dim))
        return y.split((self.heads, self.kv_heads, self.kv_heads), dim=-2)

    def _apply(self, fn, recurse=True):
        freqs = self.freqs                                        # (64 bits also where the block is cast)
        super()._apply(fn, recurse)
        if freqs is not None and self.freqs.dtype != freqs.dtype:
            self.freqs = freqs.to(self.freqs.device)
        return self

    def _positions(self, positions: torch.Tensor | None, *lead: int) -> torch.Tensor | None:
        """The positions of tokens [*lead] as the cache takes them; ValueError where they do not fit the block."""
        if (positions is None) != (self.freqs is None):
            raise ValueError("a block with frequencies needs its tokens' positions" if positions is None
                             else "positions were given to a block without frequencies")
        if positions is None:
            return None
        axes = () if self.sections is None or len(self.sections) == 1 else (len(self.sections),)
        flat = (math.prod(lead), *axes)
        if tuple(positions.shape) not in ((*lead, *axes), flat) or positions.dtype not in (torch.int32, torch.int64, torch.float32):
            raise ValueError(f"positions {tuple(positions.shape)} of {positions.dtype}: int32, int64 or float32 {(*lead, *axes)} expected")
        if positions.device != self.freqs.device:
            raise ValueError(f"positions on {positions.device}, the block's frequencies on {self.freqs.device}")
        return positions.reshape(flat)

    def _store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: Mx4KVCache, slots: torch.Tensor,
               positions: torch.Tensor | None) -> torch.Tensor:
        """Keys and values [T, kv_heads, D] into the cache; the queries [T, heads, D] to attend with."""
        if positions is None:
            cache.append(k, v, slots)
            return q
        return cache.append_rope(q, k, v, slots, positions, self.freqs, self.sections, self.interleaved)

    def forward(self, x: torch.Tensor, cache: Mx4KVCache, slots: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, positions: torch.Tensor | None = None, tree_mask: torch.Tensor | None = None,
                tree_lens: torch.Tensor | None = None) -> torch.Tensor:
        """x [B, T, hidden]: the newest T tokens of B sequences, whose slots (int64 [B * T]),
        pages and lengths (the new tokens included) are given, and with frequencies their
        positions [B, T] (several sections: [B, T, axes]). Few tokens a sequence (decoding,
        drafts to verify): every query row is read against the cache as it is stored. With
        tree_mask (and tree_lens) the tokens are a tree's nodes, as in
        ``convrot_mx4_tree_attention``; slots of padding behind them are -1."""
        b, t, _ = x.shape
        if tree_lens is not None and tree_mask is None:
            raise ValueError("tree_lens were given without a tree_mask")
        positions = self._positions(positions, b, t)
        q = self._store(*self.project(x.flatten(0, 1)), cache, slots, positions).unflatten(0, (b, t))
        if tree_mask is not None:
            y = cache.attend_tree(q, block_table, seq_lens, tree_mask, tree_lens)
        else:
            y = cache.attend(q, block_table, seq_lens)
        return self.out(y.reshape(b, t, self.heads * self.head_dim))

    def prefill(self, x: torch.Tensor, cache: Mx4KVCache, seq: int, positions: torch.Tensor | None = None) -> torch.Tensor:
        """x [T, hidden]: the next T tokens of one sequence. Many query rows: the keys and values
        so far are read back once and torch's attention runs on them. Positions of a block with
        frequencies: [T(, axes)], or None for the tokens' places in the sequence on one axis."""
        t = x.shape[0]
        device = x.device
        if positions is None and self.freqs is not None and (self.sections is None or len(self.sections) == 1):
            positions = torch.arange(cache.length(seq), cache.length(seq) + t, device=device)
        positions = self._positions(positions, t)
        q, k, v = self.project(x)
        new = torch.tensor(cache.extend(seq, t), dtype=torch.int64, device=device)
        try:
            q = self._store(q, k, v, cache, new, positions)
            ks, vs = cache.read(torch.tensor(cache.slots(seq), dtype=torch.int64, device=device), x.dtype)
            n = ks.shape[0]
            seen = torch.ones(t, n, dtype=torch.bool, device=device).tril(n - t)
            y = torch.nn.functional.scaled_dot_product_attention(
                q.transpose(0, 1)[None], ks.transpose(0, 1)[None], vs.transpose(0, 1)[None], attn_mask=seen, enable_gqa=True)
            return self.out(y[0].transpose(0, 1).reshape(t, self.heads * self.head_dim))
        except BaseException:
            cache.accept(seq, t, ())                              # (the new tokens' slots are given back)
            raise
