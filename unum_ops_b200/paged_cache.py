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

Serving only: there is no backward pass, and inputs that ask for one are refused.
"""
from __future__ import annotations

import torch

from . import _lib
from .infllm_v2 import _as_i32

__all__ = ["append_cache", "paged_attention", "evict_cache"]

_CACHE_DTYPES = (torch.bfloat16, torch.float16)


def _run(dev, fn, *args):
    if torch.cuda.current_device() == dev.index:
        _lib.check(fn(*args))
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(*args))


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise NotImplementedError("the paged cache's operators have no backward pass: call them under torch.no_grad()")


def _strides(t):
    """The strides of a 3-d tensor's first two dims, 0 for a dim of one element (whose stride says nothing)."""
    (n, m, _), (a, b, _) = t.shape, t.stride()
    return a if n > 1 else 0, b if m > 1 else 0


def _has_rows16(t):
    """Whether 16-byte loads can read the rows of a 3-d tensor of 2-byte elements."""
    a, b = _strides(t)
    return t.stride(2) == 1 and not (a | b) % 8 and not t.data_ptr() % 16


def _rows16(t):
    return t if _has_rows16(t) else t.clone(memory_format=torch.contiguous_format)


def _check_cache(k_cache, v_cache):
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 3:
            raise ValueError(f"{name} must be [n_tokens, Hk, D]; got {tuple(c.shape)}")
        if c.dtype not in _CACHE_DTYPES:
            raise ValueError(f"{name} must be bfloat16 or float16; got {c.dtype}")
        if not _has_rows16(c):
            raise ValueError(f"{name} must have contiguous, 16-byte aligned rows (strides {tuple(c.stride())})")
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"k_cache and v_cache differ: {tuple(k_cache.shape)} {k_cache.dtype} and "
                         f"{tuple(v_cache.shape)} {v_cache.dtype}")


def _overlaps(t):
    """Whether two elements of ``t`` may share memory (an expanded or an overlapping view)."""
    reach = 0
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if stride <= reach:
            return True
        reach += (size - 1) * stride
    return False


def _check_table(block_table, page_size):
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, n_pages]; got {tuple(block_table.shape)}")
    if page_size < 1 or page_size & (page_size - 1) or page_size > 65536:
        raise ValueError(f"page_size must be a power of two up to 65536; got {page_size}")
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    return bt if bt.stride(1) == 1 or bt.shape[1] < 2 else bt.contiguous()


def append_cache(k, v, k_cache, v_cache, block_table, token_to_bs, token_pos_in_bs, *, page_size=1):
    """Write new tokens' keys and values to their places in the cache, in place.

    k, v             [T, Hk, D] of the cache's dtype (any strides)
    block_table      int32 [B, n_pages]
    token_to_bs      int32 [T], the tokens' sequences
    token_pos_in_bs  int32 [T], as for get_block_table: token t sees that many positions,
                     the last of them its own, so it is written to position
                     ``token_pos_in_bs[t] - 1``
    A token whose sequence is outside [0, B), whose position is outside the table or whose
    table entry is outside the cache is not written; every other row of the cache is left as
    it was.  The tokens' places must differ from each other: where two are the same, the row
    holds pieces of either.  Returns (k_cache, v_cache)."""
    dev = _lib.require_cuda(k, v, k_cache, v_cache, block_table, token_to_bs, token_pos_in_bs)
    _no_grad(k, v, k_cache, v_cache)
    _check_cache(k_cache, v_cache)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != k_cache.shape[1:]:
        raise ValueError(f"k and v must be [T, {k_cache.shape[1]}, {k_cache.shape[2]}] like the cache's rows; got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        raise ValueError(f"k and v must have the cache's dtype {k_cache.dtype}; got {k.dtype} and {v.dtype}")
    if _overlaps(k_cache) or _overlaps(v_cache) or (k_cache.data_ptr() == v_cache.data_ptr() and k_cache.numel()):
        raise ValueError("k_cache and v_cache are written to: their rows must not share memory")
    T, Hk, D = k.shape
    if token_to_bs.numel() != T or token_pos_in_bs.numel() != T:
        raise ValueError(f"token_to_bs and token_pos_in_bs must have one entry for each of {T} tokens; got "
                         f"{token_to_bs.numel()} and {token_pos_in_bs.numel()}")
    bt = _check_table(block_table, page_size)
    if T == 0 or k.numel() == 0:
        return k_cache, v_cache
    k, v, tb, pos = _rows16(k), _rows16(v), _as_i32(token_to_bs), _as_i32(token_pos_in_bs)
    _run(dev, _lib.load().unum_cache_append, k.data_ptr(), v.data_ptr(), T, Hk, D, *_strides(k), *_strides(v),
         k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0], *_strides(k_cache), *_strides(v_cache),
         bt.data_ptr(), bt.shape[0], bt.shape[1], bt.stride(0), page_size, tb.data_ptr(), pos.data_ptr(), _lib.stream_ptr(dev))
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
                 holds): sizes the launch and, with ``weights``, its workspace
    weights      float32 [B, Hk, W >= max_seqlen], updated in place: weights[b, g, p] grows by
                 the softmax weights that the group's G heads give position p; positions
                 that are not attended to keep their value.  ``evict_cache`` reads them
    Returns [B, Hq, D] of q's dtype:
        out[b, h] = sum_p softmax_p(q[b, h] . k[token(p), h // G] * scale) v[token(p), h // G]
    over the positions whose token lies in the cache; with ``return_lse`` also the float32
    [B, Hq] natural logarithm of the softmax's sum.  A row without such a position is 0 with
    lse = -inf, and so is one whose scores are all -inf."""
    dev = _lib.require_cuda(q, k_cache, v_cache, block_table, seqlens, weights)
    _check_cache(k_cache, v_cache)
    if q.dim() != 3 or q.shape[2] != k_cache.shape[2]:
        raise ValueError(f"q must be [B, Hq, {k_cache.shape[2]}]; got {tuple(q.shape)}")
    _no_grad(q, k_cache, v_cache, *(() if weights is None else (weights,)))
    B, Hq, D = q.shape
    n_tokens, Hk = k_cache.shape[0], k_cache.shape[1]
    if q.dtype != k_cache.dtype:
        raise ValueError(f"q must have the cache's dtype {k_cache.dtype}; got {q.dtype}")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} kv heads")
    bt = _check_table(block_table, page_size)
    if bt.shape[0] != B or seqlens.numel() != B:
        raise ValueError(f"block_table and seqlens must have one row for each of {B} sequences; got {bt.shape[0]} and "
                         f"{seqlens.numel()}")
    held = bt.shape[1] * page_size
    max_seqlen = held if max_seqlen is None else min(int(max_seqlen), held)
    if max_seqlen < 0:
        raise ValueError(f"max_seqlen must not be negative; got {max_seqlen}")
    w_ptr = w_sb = w_sh = 0
    if weights is not None:
        if weights.dim() != 3 or weights.shape[:2] != (B, Hk) or weights.shape[2] < max_seqlen:
            raise ValueError(f"weights must be [{B}, {Hk}, >= {max_seqlen}]; got {tuple(weights.shape)}")
        if weights.dtype != torch.float32 or weights.stride(2) != 1 or _overlaps(weights):
            raise ValueError("weights must be float32 with contiguous rows that share no memory")
        w_ptr, w_sb, w_sh = weights.data_ptr(), weights.stride(0), weights.stride(1)
    if softmax_scale is None:
        softmax_scale = D ** -0.5
    out = torch.empty(B, Hq, D, dtype=q.dtype, device=dev)
    lse = torch.empty(B, Hq, dtype=torch.float32, device=dev) if return_lse else None
    if B:
        q, sl = _rows16(q), _as_i32(seqlens)
        L = _lib.load()
        nbytes = L.unum_paged_attention_workspace_size(B, Hq, Hk, D, max_seqlen, int(weights is not None))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)  # a call's own: calls on other streams may overlap
        _run(dev, L.unum_paged_attention, q.data_ptr(), B, Hq, D, *_strides(q), k_cache.data_ptr(),
             v_cache.data_ptr(), _lib.DTYPE_CODES[q.dtype], n_tokens, Hk, *_strides(k_cache), *_strides(v_cache),
             bt.data_ptr(), bt.shape[1], bt.stride(0), page_size, sl.data_ptr(),
             max_seqlen, float(softmax_scale), out.data_ptr(), _lib.ptr(lse), w_ptr, w_sb, w_sh, ws.data_ptr(), nbytes,
             _lib.stream_ptr(dev))
    return (out, lse) if return_lse else out


def evict_cache(block_table, seqlens, weights, *, budget, init_pages=0, local_pages=1, page_size=1):
    """Shorten each sequence's cache to ``budget`` pages, by the attention weight that its positions gathered.

    block_table  int32 [B, n_pages]
    seqlens      int32 [B], positions held (clamped to the table)
    weights      float32 [B, Hk, n_pages * page_size], as ``paged_attention`` gathers them
    Of a sequence's ceil(seqlens[b] / page_size) pages in use the first ``init_pages``, the
    last ``local_pages`` (at least one) and the heaviest others stay, ``budget`` in all, in
    their order; a sequence that has no more than that keeps them all.  A page's weight is the
    sum of its positions' weights over all kv heads, in 64 bits and rounded to 32 once; ties
    stay by the lower index and a NaN ranks below every number.
    Returns new tensors (block_table, seqlens, weights, evicted):
        block_table  the rows without the evicted pages (entries behind the pages in use move up
                     too), -1 at the end
        seqlens      less page_size for each evicted page
        weights      moved along with their pages, 0 behind the new lengths
        evicted      int32 [B, n_pages]: the evicted entries in their order, then -1: what the
                     caller's allocator gets back
    Keys and values stay where they are."""
    dev = _lib.require_cuda(block_table, seqlens, weights)
    _no_grad(weights)
    bt = _check_table(block_table, page_size)
    B, n_pages = bt.shape
    if seqlens.numel() != B:
        raise ValueError(f"seqlens must have one entry for each of {B} sequences; got {seqlens.numel()}")
    if weights.dim() != 3 or weights.shape[0] != B or weights.shape[1] < 1 or weights.shape[2] != n_pages * page_size:
        raise ValueError(f"weights must be [{B}, Hk, {n_pages * page_size}]; got {tuple(weights.shape)}")
    if weights.dtype != torch.float32:
        raise ValueError(f"weights must be float32; got {weights.dtype}")
    if local_pages < 1 or init_pages < 0 or budget < init_pages + local_pages:
        raise ValueError(f"need init_pages >= 0, local_pages >= 1 and budget >= their sum; got budget {budget}, "
                         f"init_pages {init_pages}, local_pages {local_pages}")
    w = weights if weights.stride(2) == 1 else weights.contiguous()
    Hk = w.shape[1]
    sl = _as_i32(seqlens)
    ids = torch.empty(2, B, n_pages, dtype=torch.int32, device=dev)
    new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    new_w = torch.empty(B, Hk, n_pages * page_size, dtype=torch.float32, device=dev)
    if B:
        _run(dev, _lib.load().unum_cache_evict, bt.data_ptr(), B, n_pages, bt.stride(0), sl.data_ptr(), w.data_ptr(),
             Hk, w.stride(0), w.stride(1), page_size, budget, init_pages, local_pages, ids[0].data_ptr(),
             new_lens.data_ptr(), new_w.data_ptr(), ids[1].data_ptr(), _lib.stream_ptr(dev))
    return ids[0], new_lens, new_w, ids[1]
