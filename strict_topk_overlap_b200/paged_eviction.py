"""Keeping a paged cache small: what each cached key is attended with, and
eviction of the tokens that received least.

``accumulate_weights`` adds the attention weight that each key receives from a
call's new tokens (prompts, pieces, drafted or single tokens), from the
log-sum-exps that ``paged_attention.attention`` returned for them. New: the
reference keeps every token.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib as L
from .paged import PagedKVCache
from .paged_append import _heads, _ints, _rows, _tokens
from .paged_attention import _most


def _slots(cache):
    """Blocks of the cache's table."""
    return cache.page_table.shape[0] // (cache.block_size // cache.page_size)


def empty_weights(cache: PagedKVCache) -> torch.Tensor:
    """Zero weights for every token slot of the cache: FP32 [Hkv, blocks, block_size], block
    block_offsets[r] + j // block_size holding the key j of request r."""
    return torch.zeros((cache.hkv, _slots(cache), cache.block_size), device=cache.k_pages.device)


def _weights(x, shape, name, index):
    """Address of a weights tensor."""
    if x.dtype is not torch.float32 or x.shape != shape or x.get_device() != index or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous FP32 [Hkv, blocks, block_size] = {shape} on the cache's device")
    return x.data_ptr()


@lru_cache(maxsize=1024)
def _workspace_bytes(device, dtype, hkv, block, dim, page, requests, tokens, hq, blocks, packed, most, longest, masks):
    """Workspace of a call, from its sizes alone (a pool address stands for any)."""
    any_pool = 256
    kv = L.PACK_KV(any_pool, any_pool, dtype, hkv, 0, block, dim, any_pool, any_pool, page, 0)
    with torch.cuda.device(device):
        return L.load().stk_accumulate_weights_workspace_bytes(kv, requests, tokens, hq, blocks, packed, most, longest,
                                                               masks)


def weights_workspace(cache: PagedKVCache, tokens, hq, *, token_offsets=None, max_tokens=None, masks=False):
    """Workspace for ``accumulate_weights`` of these sizes (``masks``: with ``kv_lo`` or ``kv_hi``)."""
    pool = cache.k_pages
    need = _workspace_bytes(pool.get_device(), L.dtype_code(pool), cache.hkv, cache.block_size, cache.dim,
                            cache.page_size, cache.requests, tokens, hq, _slots(cache), token_offsets is not None,
                            _most(max_tokens, tokens, token_offsets), cache.max_blocks * cache.block_size, masks)
    return torch.empty((need,), device=pool.device, dtype=torch.uint8)


def accumulate_weights(weights, q, cache: PagedKVCache, lengths, lse, *, token_offsets=None, max_tokens=None, kv_lo=None,
                       kv_hi=None, softcap=0.0, slopes=None, scale=None, workspace=None):
    """Add to ``weights`` (``empty_weights``), in place, what the packed tokens
    q [T, Hq, D] attend each key with: the sum over the tokens that see it and
    over the query heads of its KV head of exp(score - lse), ``lse`` FP32
    [T, Hq] as ``attention(..., return_lse=True)`` returned it for the same
    tokens, lengths and options. To weigh by a request's last tokens alone, pass
    those: like in ``attention``, they are the last ones of ``lengths[r]``. A
    token that sees no key (lse = -inf) adds nothing; tokens from
    token_offsets[R] on are padding. Returns ``weights``."""
    pool = cache.k_pages
    pages, hkv, _, d = pool.shape
    dtype, index = pool.dtype, pool.get_device()
    kv = cache.packed_kv(hkv, d)
    requests, blocks, block = cache.block_offsets.shape[0] - 1, _slots(cache), cache.block_size
    t, hq = _heads(q, hkv)
    qp, qt, qh = _rows(q, (t, hq, d), "q", dtype, index)
    held = _ints(lengths, (requests,), "lengths", index)
    offsets = _tokens(token_offsets, t, requests, index)
    to = _weights(weights, (hkv, blocks, block), "weights", index)
    if lse.dtype is not torch.float32 or lse.shape != (t, hq) or lse.get_device() != index or not lse.is_contiguous():
        raise ValueError("lse must be contiguous FP32 [T, Hq] on the cache's device")
    most, longest = _most(max_tokens, t, token_offsets), cache.max_blocks * block
    options, masks = None, kv_lo is not None or kv_hi is not None
    if softcap or slopes is not None or scale is not None or masks:
        if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (hq,) or
                                   slopes.get_device() != index or not slopes.is_contiguous()):
            raise ValueError("slopes must be contiguous FP32 [Hq] on the cache's device")
        if softcap < 0 or (scale is not None and scale <= 0):
            raise ValueError("softcap must not be negative and scale must be positive")
        options = L.PACK_OPTIONS(scale or 0.0, softcap, 0 if slopes is None else slopes.data_ptr(),
                                 0 if kv_lo is None else _ints(kv_lo, (t,), "kv_lo", index),
                                 0 if kv_hi is None else _ints(kv_hi, (t,), "kv_hi", index))
    if workspace is None:
        need = _workspace_bytes(index, L.dtype_code(pool), hkv, block, d, cache.page_size, requests, t, hq, blocks,
                                offsets is not None, most, longest, masks)
        if need:
            workspace = q.new_empty((need,), dtype=torch.uint8)
    else:
        if workspace.get_device() != index:
            raise ValueError("workspace must be on the cache's device")
        need = workspace.numel()
    rc = L.on_device(index, L.load().stk_accumulate_weights, kv, pages, qp, qt, qh, requests, t, hq, blocks, held, offsets,
                     most, longest, options, lse.data_ptr(), to, L.ptr(workspace), need, L.status_ptr(),
                     L.raw_stream(index))
    if rc:
        L.check(rc, "accumulate_weights")
    return weights
