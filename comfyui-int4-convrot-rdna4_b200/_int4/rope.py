"""Rotary positions for queries and keys, on one axis (text) or several (images, video).

    rope_freqs(sections, theta) -> freqs
    apply_rope(x, positions, freqs, sections, interleaved, inverse) -> x turned

Forward only, like the other operators. The rotation is orthogonal: ``inverse=True``
turns back, which is the gradient of ``apply_rope`` by x as well.
"""
from __future__ import annotations

import torch

from . import mx4


def rope_freqs(sections: int | tuple[int, ...], theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """theta^(-i / n) for the n pairs of each axis, float64 [pairs of all axes]. (A model's own scaling
    of the frequencies is applied to them by the caller.)"""
    sections = (sections,) if isinstance(sections, int) else tuple(sections)
    if not sections or min(sections) < 0:
        raise ValueError(f"sections must be numbers of pairs, got {sections}")
    return torch.cat([theta ** (-torch.arange(n, dtype=torch.float64) / max(1, n)) for n in sections]).to(device)


def apply_rope(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, sections: tuple[int, ...] | None = None,
               interleaved: bool = True, inverse: bool = False) -> torch.Tensor:
    """Turns the heads x [..., H, D] by their tokens' positions; returns a new tensor in x's dtype.

    Pair i of a head is channels (2i, 2i + 1) where ``interleaved``, else (i, i + P), of P
    pairs; channels behind the 2P first are copied. Its angle is position times
    freqs[i] (float64 [P], radians a position). sections: pairs of each position axis,
    adding up to P (None: one axis). positions int32, int64 or float32, broadcast to x's
    leading sizes [...], with several sections to [..., axes]. Angles are taken in 64 bits.

    ``convrot_mx4_cache_append_rope`` and the layers on it have ``interleaved=False`` by default: name
    the order where queries and keys go through both.

    x float32, bfloat16 or float16, any strides but a contiguous D (with more than two
    leading sizes a copy is made where they are not one stride); q and k as heads of one
    tensor take one launch.
    """
    return (mx4._native or mx4.native()).rope(x, positions, freqs, sections, interleaved, inverse)
