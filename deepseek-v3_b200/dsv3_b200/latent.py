"""The latent cache of MLA in 8 bits, and the attention that reads it.

``MLA.forward`` of the reference (model.py:396-497) keeps 512 normalised latent values and 64 rotated ones of every token in
bf16 and reads them twice per step with ``einsum``.  Here a cached token is 512 e4m3 values with one power-of-two scale
and 64 bf16 values held divided by it (644 bytes instead of 1152), tokens lie in pages of a pool that many sequences share, and the
attention multiplies the 8-bit values as they lie in the cache.

    cache = allocate_latent_cache(n_pages)
    latent_cache_write(cache, wkv_a(x), kv_norm.weight, freqs_cis, positions, slots)      # new tokens
    out = latent_attention(q_latent, q_rope, cache, block_table, seq_lens, softmax_scale)  # one token, a chain or a chunk per sequence
    out = latent_attention(..., tree_mask=mask)                                            # a tree of drafted tokens
    latent_cache_keep(cache, block_table, first, path, count)                              # its accepted branch closes ranks
    latent, rope = latent_cache_read(cache, block_table, cu_seqlens, total)                # back in bf16

Lengths, tables and masks are device memory and nothing is read back: a step can be captured in a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._lib import host

LATENT_DIM, ROPE_DIM = 512, 64


class LatentCache(NamedTuple):
    """The planes of a pool of pages.  ``page_size`` is a power of two from 16 on; token ``i`` of page ``p`` is slot ``p * page_size + i``."""
    latent: torch.Tensor        # float8_e4m3fn [pages, page_size, 512]: latent / scale
    rope: torch.Tensor          # bfloat16 [pages, page_size, 64]: rotated key / scale
    scale: torch.Tensor         # float32 [pages, page_size]: least power of two with max(amax |latent|, 1e-4) <= 448 scale


def allocate_latent_cache(n_pages: int, page_size: int = 64, device="cuda") -> LatentCache:
    """A pool whose tokens are all zero."""
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two from 16 on")
    return LatentCache(torch.zeros(n_pages, page_size, LATENT_DIM, dtype=torch.float8_e4m3fn, device=device),
                       torch.zeros(n_pages, page_size, ROPE_DIM, dtype=torch.bfloat16, device=device),
                       torch.ones(n_pages, page_size, dtype=torch.float32, device=device))


def latent_cache_write(cache: LatentCache, kv: torch.Tensor, norm_weight: torch.Tensor, freqs_cis: torch.Tensor, positions: torch.Tensor,
                       slots: torch.Tensor, eps: float = 1e-6) -> None:
    """Norm, rotation and quantisation of new tokens into their slots (model.py:469-471, 484-485).

    ``kv`` bf16 ``[..., 576]`` is the output of ``wkv_a``: 512 latent values, which get ``kv_norm`` (RMS norm with ``norm_weight``, bf16 or fp32),
    and 64 to rotate by ``freqs_cis[positions]`` (complex64 ``[n, 32]``, neighbouring values a pair).  ``positions`` and ``slots`` are int64, one per
    token, the slots all different; a token whose slot lies outside the pool (-1) is not stored.  Arithmetic in fp32, rounded once.
    A token with a value that is not finite, or at a position that the table does not hold, is stored as NaN as a whole."""
    host.latent_write(cache[0], cache[1], cache[2], kv, norm_weight, freqs_cis, positions, slots, eps)


def latent_cache_read(cache: LatentCache, block_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``cu_seqlens[b + 1] - cu_seqlens[b]`` tokens of every sequence, packed: bf16 ``[total, 512]`` and ``[total, 64]``.

    ``block_table`` int32 ``[sequences, pages]``, ``cu_seqlens`` int32 ``[sequences + 1]``; ``total`` sizes the result, whose rows at and beyond
    ``cu_seqlens[-1]`` are not written.  Tokens of a page that is none of the pool are zero."""
    return host.latent_read(cache[0], cache[1], cache[2], block_table, cu_seqlens, total)


def latent_cache_keep(cache: LatentCache, block_table: torch.Tensor, first: torch.Tensor, path: torch.Tensor, count: torch.Tensor) -> None:
    """After drafted tokens were verified: draft ``path[b, j]`` of sequence ``b`` moves to position ``first[b] + j``, for ``j < count[b]``.

    ``first`` int32 ``[sequences]``: tokens before the drafts; ``path`` int32 ``[sequences, drafts]``, strictly ascending in its first
    ``count[b]`` entries, as a path down a tree is whose nodes are numbered parents first."""
    host.latent_keep(cache[0], cache[1], cache[2], block_table, first, path, count)


def latent_attention(q_latent: torch.Tensor, q_rope: torch.Tensor, cache: LatentCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     softmax_scale: float, cu_seqlens_q: Optional[torch.Tensor] = None, tree_mask: Optional[torch.Tensor] = None,
                     return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of absorbed queries over the cache (model.py:486-494): bf16 of ``q_latent``'s shape, and with ``return_lse`` the natural logarithms
    of the softmax sums, fp32.

    ``q_latent`` bf16 ``[tokens, heads, 512]`` (``q_nope`` times ``wkv_b``'s key half) and ``q_rope`` ``[tokens, heads, 64]``, rotated, or both with the
    sequences in front (``[sequences, tokens, heads, ...]``); strides of tokens and heads are free.  ``seq_lens`` int32 ``[sequences]`` counts a sequence's cached
    tokens, those of its queries among them, which are the last ones.  ``cu_seqlens_q`` int32 ``[sequences + 1]`` for sequences with different numbers
    of queries.  Without ``tree_mask`` a query sees itself and all tokens before it; with it (int64, a word per query) all tokens before its
    sequence's queries, and of those the ones whose bit is set: at most 64 queries to a sequence.  A query that sees nothing gives zeros and -inf."""
    return host.latent_attention(q_latent, q_rope, cache[0], cache[1], cache[2], block_table, seq_lens, softmax_scale, cu_seqlens_q, tree_mask,
                                 return_lse)
