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

import torch

from . import _lib as L
from .paged import PagedKVCache
from .paged_append import _check_ints, _check_rows


def _most(max_tokens, tokens, token_offsets):
    """Bound on a request's new tokens."""
    if token_offsets is None:
        return min(1, tokens)
    return tokens if max_tokens is None else min(int(max_tokens), tokens)


def attention_workspace(cache: PagedKVCache, tokens, hq, *, token_offsets=None, max_tokens=None, prefix=0):
    """Workspace for ``attention`` (or, with ``prefix``, ``shared_prefix_attention``) of up to these sizes."""
    need = L.load().stk_paged_attention_workspace_bytes(cache.kv(), cache.requests, tokens, hq,
                                                        int(token_offsets is not None),
                                                        _most(max_tokens, tokens, token_offsets),
                                                        cache.max_blocks * cache.block_size, prefix)
    return torch.empty((need,), device=cache.k_pages.device, dtype=torch.uint8)


def _attend(q, cache, lengths, token_offsets, max_tokens, kv_lo, kv_hi, softcap, slopes, scale, return_lse, workspace,
            prefix):
    pool, requests = cache.k_pages, cache.requests
    dev = pool.device
    hq = q.shape[1] if q.ndim == 3 else 0
    _check_rows(q, cache, hq, "q")
    t = q.shape[0]
    if hq == 0 or hq % cache.hkv:
        raise ValueError("query heads must be a multiple of KV heads")
    _check_ints(lengths, (requests,), "lengths", dev)
    if token_offsets is not None:
        _check_ints(token_offsets, (requests + 1,), "token_offsets", dev)
    elif t != requests:
        raise ValueError("without token_offsets there must be one token per request")
    for name, x in (("kv_lo", kv_lo), ("kv_hi", kv_hi)):
        if x is not None:
            _check_ints(x, (t,), name, dev)
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.shape != (hq,) or slopes.device != dev or
                               not slopes.is_contiguous()):
        raise ValueError("slopes must be contiguous FP32 [Hq] on the cache's device")
    if softcap < 0 or (scale is not None and scale <= 0):
        raise ValueError("softcap must not be negative and scale must be positive")
    longest, most = cache.max_blocks * cache.block_size, _most(max_tokens, t, token_offsets)
    if t and most < 1:
        raise ValueError("max_tokens must be positive")
    if prefix < 0 or prefix % cache.page_size or prefix > longest:
        raise ValueError(f"prefix must be whole pages of {cache.page_size} tokens, at most {longest} tokens")
    out = torch.empty((t, hq, q.shape[2]), dtype=q.dtype, device=dev)
    lse = torch.empty((t, hq), dtype=torch.float32, device=dev) if return_lse else None
    lib, kv = L.load(), cache.kv()
    if workspace is None:
        need = lib.stk_paged_attention_workspace_bytes(kv, requests, t, hq, int(token_offsets is not None), most, longest,
                                                       prefix)
        workspace = torch.empty((need,), device=dev, dtype=torch.uint8)
    options = L.StkAttentionOptions(scale or 0.0, softcap, L.ptr(slopes), L.ptr(kv_lo), L.ptr(kv_hi))
    rc = lib.stk_paged_attention(kv, pool.shape[0], q.data_ptr(), q.stride(0), q.stride(1), requests, t, hq,
                                 lengths.data_ptr(), L.ptr(token_offsets), most, longest, prefix, options,
                                 out.data_ptr(),
                                 L.ptr(lse), workspace.data_ptr(), workspace.numel(), L.status_ptr(), L.stream_of(q))
    L.check(rc, "paged attention")
    return (out, lse) if return_lse else out


def attention(q, cache: PagedKVCache, lengths, *, token_offsets=None, max_tokens=None, kv_lo=None, kv_hi=None,
              softcap=0.0, slopes=None, scale=None, return_lse=False, workspace=None):
    """Attention of packed tokens q [T, Hq, D], the last ones of their requests,
    over the ``lengths[r]`` (int32 [R]) tokens that the cache holds of each:
    request r's tokens are token_offsets[r] .. token_offsets[r + 1] (int32
    [R + 1]; None: one token per request), at most ``max_tokens`` of them
    (None: T). ``kv_lo`` / ``kv_hi`` int32 [T] bound each token's keys (None:
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
