"""Paged key/value cache in e4m3 with one scale per page and head: append and attention
(the bf16 paged decode it stands beside: examples/flash_decoding/example_gqa_decode.py).

A pool of pages serves all sequences; ``block_table[b, n]`` is the page that holds the tokens
``n * page_size ..`` of sequence b, and ``lengths[b]`` counts its tokens, the new ones among them: the same
``lengths`` go to the append and to the attention of one step, where the L new tokens take the positions
``lengths[b] - L .. lengths[b] - 1``.  Positions below zero are padding (prompts of uneven length, padded on the
left): they are not stored, and their queries give zeros.

The layout is made for the attention kernel (csrc/ops/kv_attention.hip): K pages are [token, dim], V pages
[dim, token], both head-major, the head padded with zeros to a multiple of 64.

* Scales are powers of two. When a new token is larger than its page's scale allows, the page's codes are scaled
  again: exactly, but for values that become subnormal in e4m3, which are rounded once more, by up to 2^-10 of the
  new scale each time. The first token of a page sets its scale anew, whatever the page held before. Scales of an
  append are 2^-22 at least; pools that a caller fills may hold V scales down to 2^-68 (a smaller one counts as
  that).
* A page that sequences share may be read by all of them; only one may append to it in a call.
* Page ids outside the pool (a table padded with -1, say) are not followed: their tokens are not stored, and count
  as absent for the attention.  So do tokens beyond the table.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from tilelang import _native


class KVCache(NamedTuple):
    """The pools of one layer."""
    k: torch.Tensor  # float8_e4m3fn [pages, kv_heads, page_size, wide]
    v: torch.Tensor  # float8_e4m3fn [pages, kv_heads, wide, page_size]
    k_scale: torch.Tensor  # float32 [pages, kv_heads]
    v_scale: torch.Tensor  # float32 [pages, kv_heads]
    head_dim: int  # wide is the next multiple of 64


def alloc_kv_cache(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> KVCache:
    """Empty pools.  ``head_dim`` up to 256; ``page_size`` a power of two from 16 to 1024."""
    if not 1 <= head_dim <= 256:
        raise ValueError(f"alloc_kv_cache: head_dim is {head_dim}, expected 1 to 256")
    if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
        raise ValueError(f"alloc_kv_cache: page_size is {page_size}, expected a power of two from 16 to 1024")
    wide = -(-head_dim // 64) * 64

    def pool(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

    return KVCache(pool(pages, kv_heads, page_size, wide), pool(pages, kv_heads, wide, page_size),
                   torch.ones(pages, kv_heads, device=device), torch.ones(pages, kv_heads, device=device), head_dim)


def kv_cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor) -> None:
    """Store the new tokens k, v [batch, L, kv_heads, head_dim] (bf16, fp16 or fp32, any strides) in place.

    ``block_table`` int32 [batch, n], ``lengths`` int32 [batch] with the new tokens counted.  Infinities are
    stored as the page's largest value, not-a-numbers as themselves; neither sets a scale.  The pools and their
    scales may share memory neither with each other nor with the call's other arguments."""
    _native.ops().kv_cache_append(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.head_dim, k, v, block_table,
                                  lengths)


def kv_cache_attention(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lengths: torch.Tensor,
                       sm_scale: Optional[float] = None,
                       return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of the L newest tokens' queries q [batch, L, heads, head_dim] (bf16 or fp16, any strides)
    over their sequences' cached tokens: query i sees the positions up to ``lengths - L + i``.

    ``heads`` is a multiple of the cache's kv_heads (consecutive query heads share one); ``sm_scale`` defaults to
    ``head_dim ** -0.5``.  Returns out as q, and with ``return_lse`` the natural logarithm of the softmax's
    denominator, float32 [batch, L, heads].  A query that sees nothing gives zeros and -inf."""
    return _native.ops().kv_cache_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.head_dim,
                                            block_table, lengths, sm_scale, return_lse)
