"""The paged key-value cache: its writes, attention of one new token over it, and its eviction.

No reference functions: the reference's get_block_table
(src/unum_ops/sparse_kernel_extension/get_table_torch.py:4-44) maps positions to
physical tokens for an attention kernel and a cache that live outside the
repository.  These operators are that cache's other half, beside
``sparse_attention``, which reads the selected blocks only.

The cache is a pair of tensors ``k_cache``, ``v_cache`` [n_tokens, Hk, D] (bf16 or
fp16, D = 64 or 128, any token and head strides that are multiples of 8 elements,
also views of one [n_tokens, 2, Hk, D] tensor).  Position p of sequence b lives at token
``block_table[b, p // page_size] * page_size + p % page_size``; ``page_size`` is a
power of two, and 1 is the table that ``get_block_table`` and ``sparse_attention``
read (the same caches serve both, with ``head_group = Hk`` there).  A table entry
outside the cache marks positions that are not held: they are neither read nor written.

Tables, lengths and ids are int32; other types are converted on the way (a kernel or two
more), and what 32 bits do not hold becomes their least or largest number: such an entry is
outside the cache, such a length above every bound.

Serving only: there is no backward pass and no forward-mode derivative, and inputs that ask
for one are refused.
"""
from __future__ import annotations

from . import _lib

__all__ = ["append_cache", "paged_attention", "evict_cache"]


def append_cache(k, v, k_cache, v_cache, block_table, token_to_bs, token_pos_in_bs, *, page_size=1):
    """Write new tokens' keys and values to their places in the cache, in place.

    k, v             [T, Hk, D] of the cache's dtype (any strides), not in the caches' memory
    block_table      int32 [B, n_pages]
    token_to_bs      int32 [T], the tokens' sequences
    token_pos_in_bs  int32 [T], as for get_block_table: token t sees that many positions,
                     the last of them its own, so it is written to position
                     ``token_pos_in_bs[t] - 1``
    A token whose sequence is outside [0, B), whose position is outside the table (or 2^31 - 2
    and more) or whose table entry is outside the cache is not written; every other row of the cache is left as
    it was.  The tokens' places must differ from each other: where two are the same, the row
    holds pieces of either.  Returns (k_cache, v_cache)."""
    _lib.binding().append_cache(k, v, k_cache, v_cache, block_table, token_to_bs, token_pos_in_bs, page_size)
    return k_cache, v_cache


def paged_attention(q, k_cache, v_cache, block_table, seqlens, *, page_size=1, max_seqlen=None, softmax_scale=None,
                    weights=None, return_lse=False):
    """Attention of one new token for each sequence over its whole cache.

    q            [B, Hq, D] of the cache's dtype, Hq = G * Hk with G <= 64
    block_table  int32 [B, n_pages]
    seqlens      int32 [B]: positions [0, seqlens[b]) are attended to (the new token's own
                 among them, once ``append_cache`` has written it); counts outside
                 [0, max_seqlen] are clamped
    max_seqlen   an upper bound of seqlens known on the host (default: what the table
                 holds): sizes the launch and, with ``weights``, its workspace of
                 B * Hq * max_seqlen * 4 bytes
    weights      float32 [B, Hk, W >= max_seqlen], updated in place: weights[b, g, p] grows by
                 the softmax weights that the group's G heads give position p; positions
                 that are not attended to keep their value.  ``evict_cache`` reads them
    Returns [B, Hq, D] of q's dtype:
        out[b, h] = sum_p softmax_p(q[b, h] . k[token(p), h // G] * scale) v[token(p), h // G]
    over the positions whose token lies in the cache; with ``return_lse`` also the float32
    [B, Hq] natural logarithm of the softmax's sum.  A row without such a position is 0 with
    lse = -inf, and so is one whose scores are all -inf."""
    return _lib.binding().paged_attention(q, k_cache, v_cache, block_table, seqlens, page_size, max_seqlen, softmax_scale,
                                          weights, return_lse)


def evict_cache(block_table, seqlens, weights, *, budget, init_pages=0, local_pages=1, page_size=1):
    """Shorten each sequence's cache to ``budget`` pages, by the attention weight that its positions gathered.

    block_table  int32 [B, n_pages]
    seqlens      int32 [B], positions held (clamped to the table)
    weights      float32 [B, Hk, n_pages * page_size], as ``paged_attention`` gathers them
    Of a sequence's ceil(seqlens[b] / page_size) pages in use the first ``init_pages``, the
    last ``local_pages`` (at least one) and the heaviest others stay, ``budget`` in all, in
    their order; a sequence that has no more than that keeps them all.  A page's weight is the
    sum of its positions' weights over all kv heads, in 64 bits and rounded to 32 once; ties
    stay by the lower index and a NaN ranks below every number.  With ``budget ==
    init_pages + local_pages`` nothing is chosen, and the weights only move along.
    Returns new tensors (block_table, seqlens, weights, evicted):
        block_table  the rows without the evicted pages (entries behind the pages in use move up
                     too), -1 at the end
        seqlens      less page_size for each evicted page
        weights      moved along with their pages, 0 behind the new lengths
        evicted      int32 [B, n_pages]: the evicted entries in their order, then -1: what the
                     caller's allocator gets back
    Keys and values stay where they are.  At most 409600 pages a sequence."""
    return _lib.binding().evict_cache(block_table, seqlens, weights, budget, init_pages, local_pages, page_size)
