"""Paged key / value caches in the caller's hands: attention of new tokens with a sliding window and first tokens that stay
visible, and eviction by the attention weight that cached tokens have received.

No counterpart in the reference, whose ``decode_once`` (layers.py:316-344) keeps the last ``seq - 1`` tokens of every sequence.
A cache is tensors on one GPU: ``kpool`` and ``vpool`` bf16 ``[n_pages, kv_heads, 64, d_head]`` (the layout of the runtime's own
caches; keys rotated by the caller), ``page_table`` int32 ``[batch, pages]`` and ``lengths`` int32 ``[batch]``, which layers of one
model can share.  Everything runs on the current stream of the tensors' GPU, allocates nothing but its results and its scratch,
reads nothing back, and can be captured into a CUDA graph.  Nothing here records gradients.
"""
from __future__ import annotations

import struct

import torch

from ._lib import MTJ_BF16, MTJ_F32, check, lib

PAGE_TOKENS = 64
_DTYPES = {torch.bfloat16: MTJ_BF16, torch.float32: MTJ_F32}
# mtj_cache_attn_args and mtj_cache_evict_args as the C side lays them out (the fields of MtjCacheAttnArgs, MtjCacheEvictArgs): a
# token's call is launched in a few microseconds, of which filling a ctypes structure would be a quarter
_ATTN_ARGS = struct.Struct("@12P4q10if4x").pack
_EVICT_ARGS = struct.Struct("@11P8i").pack
_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
# tensors are asked for the number of their GPU (-1: the host's memory), which costs less than for their device


def _want(t, name, dtype, shape, index):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on cuda:{index}")


def _pool_shape(kpool, vpool, page_table, lengths):
    shape = kpool.shape if isinstance(kpool, torch.Tensor) else ()
    if len(shape) != 4 or shape[2] != PAGE_TOKENS or not kpool.is_cuda or kpool.dtype != _BF16 or not kpool.is_contiguous():
        raise ValueError(f"kpool must be a contiguous bfloat16 CUDA tensor [n_pages, kv_heads, {PAGE_TOKENS}, d_head]")
    table = page_table.shape if isinstance(page_table, torch.Tensor) else ()
    index = kpool.get_device()
    if len(table) != 2 or page_table.dtype != _I32 or page_table.get_device() != index or not page_table.is_contiguous():
        raise ValueError(f"page_table must be a contiguous int32 tensor [batch, pages] on cuda:{index}")
    _want(vpool, "vpool", _BF16, shape, index)
    _want(lengths, "lengths", _I32, table[:1], index)
    return shape, table, index


def _like(t, name, shape, dtype, index):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != index or t.shape != shape:
        raise ValueError(f"{name} must be a {dtype} tensor {list(shape)} on cuda:{index}")


def _rows(t, shape):
    """``t`` [batch, tokens, heads, d_head] with heads side by side in a row, rows at one stride and 16-byte aligned (a slice
    of a fused projection is one); anything else is copied."""
    at = t.data_ptr()
    if t.is_contiguous():
        if at & 15:
            t = t.clone()
            at = t.data_ptr()
        return t, at, shape[2] * shape[3]
    s, (batch, tokens, heads, d_head) = t.stride(), shape
    ld = s[1] if tokens > 1 else s[0] if batch > 1 else heads * d_head
    if s[3] == 1 and (s[2] == d_head or heads == 1) and ld >= heads * d_head and not ld & 7 and not at & 15 and \
            (batch == 1 or s[0] == ld * tokens):
        return t, at, ld
    t = t.contiguous()
    return t, t.data_ptr(), heads * d_head


def cache_attention(q, k, v, kpool, vpool, page_table, lengths, new=None, window=None, sinks=0, scale=None, weights=None,
                    weights_out=None, out=None, status=None):
    """Appends the new tokens' keys and values to the cache and attends from them over it.

    ``q`` [batch, tokens, heads, d_head] bf16 or float32; ``k``, ``v`` [batch, tokens, kv_heads, d_head] of the same type, or both
    None when the cache holds them already.  ``lengths`` counts the slots in use with the new tokens; ``new`` int32 [batch] says
    how many of the ``tokens`` rows of each sequence are new ones (default: all).  Token t of sequence b sits in slot
    ``p = lengths[b] - new[b] + t`` and sees slot j when ``j <= p and (j < sinks or p - j < window)`` (``window`` None: all).
    Slots that no new token sees are not looked at: they may hold anything, and pages of nothing else need not exist.
    Scores are multiplied by ``scale`` (default ``d_head ** -0.5``).  Returns ``out`` like ``q``; rows from ``new[b]`` on are zeros.

    ``weights`` float32 [batch, kv_heads, pages * 64]: the attention weight that each slot receives, summed over the tokens and
    over the query heads that read its head, is added to it, slots of new tokens beginning at zero.  With ``weights_out`` the
    sums go there and ``weights`` (may be None: zeros) stays as it is.
    What drafted tokens add to older slots is not taken back with their own slots.  Weights of taken tokens alone: attend without, check the drafts,
    and call again with the lengths as they are then, ``new`` the number taken plus one, the same ``q`` and no ``k`` and ``v``.

    ``out`` [batch, tokens, heads, d_head], if given, is written instead of a new tensor.  It shares no memory with the others,
    nor do ``weights`` and ``weights_out`` unless they are the same.

    ``status`` int32 [1], if given, collects what the GPU found wrong: bit 1 a length or a page number outside the cache (that
    sequence counts as empty, that page as unseen), bit 0 a wait that ran out."""
    (n_pages, kv_heads, _, d_head), (batch, pages), index = _pool_shape(kpool, vpool, page_table, lengths)
    shape = q.shape if isinstance(q, torch.Tensor) else ()
    of_q = q.dtype if len(shape) == 4 else None
    dtype = _DTYPES.get(of_q)
    if dtype is None or q.get_device() != index or shape[0] != batch or shape[3] != d_head or shape[1] < 1 or shape[2] < 1:
        raise ValueError(f"q must be a bfloat16 or float32 tensor [{batch}, tokens, heads, {d_head}] on cuda:{index}")
    _, tokens, heads, _ = shape
    q, at_q, ld_q = _rows(q, shape)
    at_k = at_v = ld_k = ld_v = 0
    if k is not None and v is not None:
        new_shape = (batch, tokens, kv_heads, d_head)
        _like(k, "k", new_shape, of_q, index)
        _like(v, "v", new_shape, of_q, index)
        k, at_k, ld_k = _rows(k, new_shape)
        v, at_v, ld_v = _rows(v, new_shape)
    elif k is not None or v is not None:
        raise ValueError("k and v come together")
    at_new = at_status = at_in = at_out = 0
    if new is not None:
        _want(new, "new", _I32, (batch,), index)
        at_new = new.data_ptr()
    if status is not None:
        _want(status, "status", _I32, (1,), index)
        at_status = status.data_ptr()
    if weights is not None or weights_out is not None:
        if weights_out is None:
            weights_out = weights
        slots = (batch, kv_heads, pages * PAGE_TOKENS)
        _want(weights_out, "weights_out", _F32, slots, index)
        at_out = weights_out.data_ptr()
        if weights is not None:
            _want(weights, "weights", _F32, slots, index)
            at_in = weights.data_ptr()
    if out is None:
        out = torch.empty(batch, tokens, heads, d_head, dtype=of_q, device=kpool.device)
        at, ld_out = out.data_ptr(), heads * d_head
    else:
        given = out
        _like(out, "out", shape, of_q, index)
        out, at, ld_out = _rows(out, shape)
        if out is not given:
            raise ValueError("out must have its heads side by side, rows at one stride and a 16-byte alignment")
    try:
        a = _ATTN_ARGS(kpool.data_ptr(), vpool.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), at_new, at_status, at_q, at_k, at_v, at,
                       at_in, at_out, ld_q, ld_k, ld_v, ld_out, n_pages, batch, pages, heads, kv_heads, d_head, tokens, dtype,
                       pages * PAGE_TOKENS if window is None else min(window, 0x7fffffff), min(sinks, 0x7fffffff),
                       d_head ** -0.5 if scale is None else scale)
    except (struct.error, OverflowError, TypeError) as e:
        raise ValueError(f"window and sinks must be whole numbers, scale a number: {e}") from None
    if index != _current_device():
        with torch.cuda.device(index):
            _run_attention(a, kpool, index)
    else:
        _run_attention(a, kpool, index)
    return out


def _run_attention(a, kpool, index):
    nbytes = lib.mtj_k_cache_attn_scratch_bytes(a)
    if nbytes < 0:
        raise ValueError(lib.mtj_last_error().decode("utf-8", "replace"))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=kpool.device)
    check(lib.mtj_k_cache_attn(a, scratch.data_ptr(), nbytes, _stream(index)))


def cache_evict(kpool, vpool, page_table, lengths, weights, spare_pages, keep, first=0, last=0, status=None):
    """Cuts every sequence that holds more than ``keep`` slots down to ``keep``: each key head keeps the ``first`` first slots, the
    ``last`` last ones and the heaviest by ``weights`` of the others (the lower slot among equals; NaN counts as heavier than any number),
    in the order of their slots.

    The kept keys and values are copied to ``spare_pages`` int32 [batch, ceil(keep / 64)], pages that no sequence uses, each
    named once.  Returns ``(kept, lengths, weights, page_table)``, new tensors: the slots that were kept [batch, kv_heads, keep]
    (-1 behind the last), and the cache as it is now.  The new table of a sequence that was cut names its spare pages, with -1
    behind them where the caller puts pages for the tokens to come; its old pages are free again.  Sequences of ``keep`` slots
    or fewer keep their pages and leave their spare ones unused."""
    (n_pages, kv_heads, _, d_head), (batch, pages), index = _pool_shape(kpool, vpool, page_table, lengths)
    keep, first, last = int(keep), int(first), int(last)
    if keep < 1 or first < 0 or last < 0 or first + last > keep:
        raise ValueError("keep must be positive and hold the first and the last slots")
    _want(weights, "weights", _F32, (batch, kv_heads, pages * PAGE_TOKENS), index)
    _want(spare_pages, "spare_pages", _I32, (batch, (keep + PAGE_TOKENS - 1) // PAGE_TOKENS), index)
    if status is not None:
        _want(status, "status", _I32, (1,), index)
    kept = torch.empty(batch, kv_heads, keep, dtype=_I32, device=kpool.device)
    lengths_out, weights_out, table_out = torch.empty_like(lengths), torch.empty_like(weights), torch.empty_like(page_table)
    a = _EVICT_ARGS(
        kpool.data_ptr(), vpool.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), weights.data_ptr(), spare_pages.data_ptr(),
        kept.data_ptr(), lengths_out.data_ptr(), weights_out.data_ptr(), table_out.data_ptr(),
        status.data_ptr() if status is not None else 0, n_pages, batch, pages, kv_heads, d_head, keep, first, last)
    if index != _current_device():
        with torch.cuda.device(index):
            check(lib.mtj_k_cache_evict(a, _stream(index)))
    else:
        check(lib.mtj_k_cache_evict(a, _stream(index)))
    return kept, lengths_out, weights_out, table_out
