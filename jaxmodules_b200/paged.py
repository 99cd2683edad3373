"""A cache of keys and values in pages, and attention over it: what a model decodes from.

The reference has no counterpart: its attention takes dense keys and values of the whole context.  A step of decoding is

    lengths += 1
    q = append_kv(cache, k, v, lengths, q=q, frequencies=f)      # [B, 1, H, d]
    o = paged_attention(q, cache, lengths)

and both calls, like ``read_kv``, can be captured into a CUDA graph (after a first call outside of one): everything that changes between steps lies
on the device.  None of the three is differentiable: tensors that require a gradient, and dual tensors of forward mode, are refused.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _native as nat
from .heads import layout_of


@dataclass(frozen=True)
class PagedCache:
    """Keys and values of many sequences in pages of ``page_size`` tokens.

    ``k``, ``v``: ``[pages, page_size, Hkv, d]``, float32 or bfloat16, d a multiple of 8 and at most 128; the strides of both alike, every head on 16 bytes.
    ``page_table``: int32 ``[B, width]``: ``page_table[b, i]`` is the page of positions ``i * page_size`` and up of sequence b; entries that no position
    reaches may be anything.  Sequences may share pages that are not written any more.  ``paged_attention`` takes up to 64 GiB of keys and as much of values.

    4 bits: ``k``, ``v`` are uint8 ``[pages, page_size, Hkv, d / 2]``, d 32, 64, 96 or 128: e2m1 codes, two to a byte, the earlier component in the lower
    half; ``k_scale``, ``v_scale`` uint8 ``[pages, page_size, Hkv, d / 32]``: every 32 components share the power of two ``2 ** (byte - 127)``, 255 is NaN.
    ``paged_attention`` takes any powers, values below 2^-100 as zeros where that is simpler; where a head's are further apart than 2^14, or its largest is not between 2^-40
    and 2^40, it takes 1.7 times as long over the rest of that sequence.
    """
    k: torch.Tensor
    v: torch.Tensor
    page_table: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, page_size: int, heads: int, d: int, page_table: torch.Tensor, dtype=torch.bfloat16) -> "PagedCache":
        """A cache of zeros on the device of ``page_table``; ``dtype``: float32, bfloat16 or ``"4bit"``."""
        zeros = lambda n, kind: [torch.zeros((pages, page_size, heads, n), dtype=kind, device=page_table.device) for _ in range(2)]
        if dtype == "4bit":
            if d % 32 or not 0 < d <= 128:
                raise ValueError("a 4-bit cache has heads of 32, 64, 96 or 128 components")
            return cls(*zeros(d // 2, torch.uint8), page_table, *zeros(d // 32, torch.uint8))
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("dtype must be float32, bfloat16 or '4bit'")
        return cls(*zeros(d, dtype), page_table)


def append_kv(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, *, new_lengths: Optional[torch.Tensor] = None,
              q: Optional[torch.Tensor] = None, frequencies: Optional[torch.Tensor] = None, layout: str = "half", magnitude: float = 1.0,
              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Optional[torch.Tensor]:
    """Writes the keys and values of new tokens into their pages, and returns the queries ready for ``paged_attention`` (None without ``q``).

    ``k``, ``v``: ``[B, T, Hkv, d]``, ``q``: ``[B, T, Hq, d]``, of the cache's dtype (float32 or bfloat16 for a 4-bit cache).  ``lengths``: int32 ``[B]``, the tokens
    of each sequence with the new ones; of the T given the first ``new_lengths[b]`` (int32, taken as at least 0 and at most T; None: all) are real and lie at positions
    ``lengths[b] - new_lengths[b]`` and up.  The others are not written, and their queries come back as zeros.

    Queries and keys are normed and rotated on the way as by ``rotate_heads``, at the positions they lie at; values are not changed.  A 4-bit
    cache takes of every 32 components the smallest power of two with which the largest is at most 6, and the nearest codes (ties to
    the even one) of the float32 results.

    Tokens at positions that the page table does not cover, or whose page is not in the cache, are not written, and
    ``attention.device_status`` reports it.  Two real tokens must not lie in one slot of one page.  Not differentiable.
    """
    return nat.host().append(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, k, v, lengths, new_lengths, q, frequencies, layout_of(layout),
                             magnitude, q_weight, k_weight, eps)


def read_kv(cache: PagedCache, lengths: torch.Tensor, max_length: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached tokens as dense keys and values ``[B, max_length, Hkv, d]`` in position order, zeros from ``lengths[b]`` on: what
    ``masked_attention_via_map`` takes, for a chunk of a prompt that attends to all before it.  In the cache's dtype, bfloat16 of a 4-bit
    cache, whose values that holds exactly (down to 2^-133).  Positions without a page read as zeros, and ``attention.device_status`` reports them.  Not differentiable."""
    return nat.host().read(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, lengths, max_length)


def paged_attention(q: torch.Tensor, cache: PagedCache, lengths: torch.Tensor, *, new_lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    window: Optional[int] = None, out_dtype: Optional[torch.dtype] = None, return_lse: bool = False):
    """Attention of the newest tokens of every sequence over the cache, themselves included: ``[B, T, Hq, d]``.

    ``q``: ``[B, T, Hq, d]``, of the cache's dtype (bfloat16 for a 4-bit cache); the heads of the cache divide Hq.  ``lengths`` and ``new_lengths`` as for
    ``append_kv``.  Token i sees the keys at its own position and before; with ``window`` only those at most ``window`` positions before.
    ``scale`` replaces ``1 / sqrt(d)``.  Rows that see no key, and tokens that are not real, are zeros, with a log-sum-exp of -inf.
    Products are summed in float32, with weights that are good to 2^-15 (bfloat16 cache) or 2^-11 (4 bits) of themselves.
    ``out_dtype`` is float32 as for ``masked_attention_via_map``, or bfloat16; ``return_lse``: also the log-sum-exp ``[B, Hq, T]``.

    Made for few new tokens: the time is that of reading the keys and values once.  For the many tokens of a prompt, ``read_kv`` and
    ``masked_attention_via_map`` use the tensor core better.  Nothing behind ``lengths[b]`` reaches a result, nor what lies outside a row's
    window or after its token, infinities and NaN included (but which values of a 4-bit cache the rows of a call see together may change their rounding).  Positions without a page make the results invalid, and ``attention.device_status``
    reports them.  Repeated calls give the same bits; a sequence in another batch need not give those.  Not differentiable.
    """
    if out_dtype is not None and out_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("out_dtype must be float32 or bfloat16")
    o, lse = nat.host().paged(cache.k, cache.v, cache.page_table, cache.k_scale, cache.v_scale, q, lengths, new_lengths, scale, window,
                              out_dtype == torch.bfloat16, return_lse)
    return (o, lse) if return_lse else o
