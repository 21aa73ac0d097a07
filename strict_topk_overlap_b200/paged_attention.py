"""Dense attention over a paged cache: prompts, pieces of prompts, drafted
tokens, single tokens, and batches behind one shared prefix.

Scores s = scale q.k may be capped (``softcap`` tanh(s / ``softcap``)) and
biased by distance (minus ``slopes[h]`` |pos - j|), in that order. A token
sees the keys kv_lo <= j < kv_hi of its request: causal by default; a sliding
window, documents packed into one request (kv_lo = the document's start) and
a prefix that sees all of itself (kv_hi = max(pos + 1, prefix)) are such
intervals too. A token that sees no key gets zeros. New: the reference attends
lists of blocks only.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib as L
from .paged import PagedKVCache
from .paged_append import _heads, _ints, _rows, _tokens


def _most(max_tokens, tokens, token_offsets):
    """Bound on a request's new tokens."""
    if token_offsets is None or tokens == 0:
        return min(1, tokens)
    if max_tokens is None:
        return tokens
    if max_tokens < 1:
        raise ValueError("max_tokens must be positive")
    return min(int(max_tokens), tokens)


@lru_cache(maxsize=1024)
def _workspace_bytes(device, dtype, hkv, block, dim, page, requests, tokens, hq, packed, most, longest, prefix):
    """Workspace of a call, from its sizes alone (a pool address stands for any)."""
    any_pool = 256
    kv = L.PACK_KV(any_pool, any_pool, dtype, hkv, 0, block, dim, any_pool, any_pool, page, 0)
    with torch.cuda.device(device):
        return L.load().stk_paged_attention_workspace_bytes(kv, requests, tokens, hq, packed, most, longest, prefix)


def attention_workspace(cache: PagedKVCache, tokens, hq, *, token_offsets=None, max_tokens=None, prefix=0):
    """Workspace for ``attention`` (or, with ``prefix``, ``shared_prefix_attention``) of these sizes."""
    pool = cache.k_pages
    need = _workspace_bytes(pool.get_device(), L.dtype_code(pool), cache.hkv, cache.block_size, cache.dim,
                            cache.page_size, cache.requests, tokens, hq, token_offsets is not None,
                            _most(max_tokens, tokens, token_offsets), cache.max_blocks * cache.block_size, prefix)
    return torch.empty((need,), device=pool.device, dtype=torch.uint8)


def _attend(q, cache, lengths, token_offsets, max_tokens, kv_lo, kv_hi, softcap, slopes, scale, return_lse, workspace,
            prefix):
    pool = cache.k_pages
    pages, hkv, _, d = pool.shape
    dtype, index = pool.dtype, pool.get_device()
    kv = cache.packed_kv(hkv, d)
    requests = cache.block_offsets.shape[0] - 1
    t, hq = _heads(q, hkv)
    qp, qt, qh = _rows(q, (t, hq, d), "q", dtype, index)
    held = _ints(lengths, (requests,), "lengths", index)
    offsets = _tokens(token_offsets, t, requests, index)
    most = _most(max_tokens, t, token_offsets)
    block, page = cache.block_size, cache.page_size
    longest = cache.max_blocks * block
    options = None
    if softcap or slopes is not None or scale is not None or kv_lo is not None or kv_hi is not None:
        if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (hq,) or
                                   slopes.get_device() != index or not slopes.is_contiguous()):
            raise ValueError("slopes must be contiguous FP32 [Hq] on the cache's device")
        if softcap < 0 or (scale is not None and scale <= 0):
            raise ValueError("softcap must not be negative and scale must be positive")
        options = L.PACK_OPTIONS(scale or 0.0, softcap, 0 if slopes is None else slopes.data_ptr(),
                                 0 if kv_lo is None else _ints(kv_lo, (t,), "kv_lo", index),
                                 0 if kv_hi is None else _ints(kv_hi, (t,), "kv_hi", index))
    if prefix and (prefix < 0 or prefix % page or prefix > longest):
        raise ValueError(f"prefix must be whole pages of {page} tokens, at most {longest} tokens")
    if workspace is None:
        need = _workspace_bytes(index, L.dtype_code(pool), hkv, block, d, page, requests, t, hq, offsets is not None,
                                most, longest, prefix)
        if need:
            workspace = q.new_empty((need,), dtype=torch.uint8)
    else:
        if workspace.get_device() != index:
            raise ValueError("workspace must be on the cache's device")
        need = workspace.numel()
    out = q.new_empty((t, hq, d))
    lse = q.new_empty((t, hq), dtype=torch.float32) if return_lse else None
    rc = L.on_device(index, L.load().stk_paged_attention, kv, pages, qp, qt, qh, requests, t, hq, held, offsets, most,
                     longest, prefix, options, out.data_ptr(), L.ptr(lse), L.ptr(workspace), need, L.status_ptr(),
                     L.raw_stream(index))
    if rc:
        L.check(rc, "paged attention")
    return (out, lse) if return_lse else out


def attention(q, cache: PagedKVCache, lengths, *, token_offsets=None, max_tokens=None, kv_lo=None, kv_hi=None,
              softcap=0.0, slopes=None, scale=None, return_lse=False, workspace=None):
    """Attention of packed tokens q [T, Hq, D], the last ones of their requests,
    over the ``lengths[r]`` (int32 [R]) tokens that the cache holds of each:
    request r's tokens are token_offsets[r] .. token_offsets[r + 1] (int32
    [R + 1]; None: one token per request; tokens from token_offsets[R] on are
    padding and get zeros), at most ``max_tokens`` of them (None: T). ``kv_lo`` / ``kv_hi`` int32 [T] bound each token's keys (None:
    causal), ``slopes`` FP32 [Hq]. Returns [T, Hq, D] in q's dtype and, with
    ``return_lse``, the log-sum-exp of each row's scores, FP32 [T, Hq]."""
    return _attend(q, cache, lengths, token_offsets, max_tokens, kv_lo, kv_hi, softcap, slopes, scale, return_lse,
                   workspace, 0)


def shared_prefix_attention(q, cache: PagedKVCache, lengths, prefix, *, token_offsets=None, max_tokens=None,
                            kv_lo=None, kv_hi=None, softcap=0.0, slopes=None, scale=None, return_lse=False,
                            workspace=None):
    """``attention`` for a batch whose requests all begin with the same
    ``prefix`` tokens (whole pages): their page tables name the same pages
    there. The prefix is read once for all requests' tokens instead of once
    per request, and joined with each request's own rest."""
    return _attend(q, cache, lengths, token_offsets, max_tokens, kv_lo, kv_hi, softcap, slopes, scale, return_lse,
                   workspace, prefix)
