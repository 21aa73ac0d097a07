"""Keeping a paged cache small: what each cached key is attended with, and
eviction of the tokens that received least.

``accumulate_weights`` adds the attention weight that each key receives from a
call's new tokens (prompts, pieces, drafted or single tokens), from the
log-sum-exps that ``paged_attention.attention`` returned for them. ``evict``
cuts requests back to a number of tokens per KV head by those weights (or any
others: they are a plain tensor), strictly, ties to the lower place like every
selection here, and leaves a cache that all other calls read: what stays moves
to the front of the requests' own pages, in its order. A kept key stays rotated
by the position it was appended with, so after an eviction append with explicit
``positions``; attention's distance ``slopes``, ``kv_lo`` and ``kv_hi`` count
places in the cache. New: the reference keeps every token.
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
    return torch.zeros((cache.hkv, _slots(cache), cache.block_size), dtype=torch.float32, device=cache.k_pages.device)


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
        if workspace.get_device() != index or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous and on the cache's device")
        need = workspace.numel()
    rc = L.on_device(index, L.load().stk_accumulate_weights, kv, pages, qp, qt, qh, requests, t, hq, blocks, held, offsets,
                     most, longest, options, lse.data_ptr(), to, L.ptr(workspace), need, L.status_ptr(),
                     L.raw_stream(index))
    if rc:
        L.check(rc, "accumulate_weights")
    return weights


def _kept(keep):
    """The number of tokens that stay, as the library takes it."""
    keep = int(keep)
    if not 1 <= keep < 2 ** 31:
        raise ValueError(f"keep = {keep} must be positive and fit into 32 bits")
    return keep


@lru_cache(maxsize=1024)
def _evict_bytes(device, dtype, hkv, block, dim, page, requests, blocks, keep, longest):
    any_pool = 256
    kv = L.PACK_KV(any_pool, any_pool, dtype, hkv, 0, block, dim, any_pool, any_pool, page, 0)
    with torch.cuda.device(device):
        return L.load().stk_evict_tokens_workspace_bytes(kv, requests, blocks, keep, longest)


def evict_workspace(cache: PagedKVCache, keep):
    """Workspace for ``evict`` down to ``keep`` tokens."""
    pool, keep = cache.k_pages, _kept(keep)
    need = _evict_bytes(pool.get_device(), L.dtype_code(pool), cache.hkv, cache.block_size, cache.dim, cache.page_size,
                        cache.requests, _slots(cache), keep, cache.max_blocks * cache.block_size)
    return torch.empty((need,), device=pool.device, dtype=torch.uint8)


def evict(cache: PagedKVCache, weights, lengths, keep, *, first=0, last=0, weights_out=None, workspace=None):
    """Cut every request that holds more than ``keep`` of ``lengths[r]`` (int32
    [R]) tokens back to ``keep``. Per KV head the ``first`` and the ``last``
    ones stay, and of the others those of the largest ``weights`` (ties to the
    lower place, NaN above all). Keys, values and weights of what stays move to
    the front, in their order; lo / hi of the blocks that changed are taken anew
    (where the cache keeps them), emptied blocks get ``empty_paged_cache``'s.
    Weights go to ``weights_out`` (None: in place; memory that overlaps
    theirs in part is refused), zeros behind the last token.
    Pages that requests share are written where their tokens move: protect a
    shared prefix by ``first``. Requests hold at most 393,216 tokens. Returns the
    new lengths [R] and the kept places [R, Hkv, keep] int32, ascending, -1
    behind a shorter request's last."""
    pool = cache.k_pages
    pages, hkv, _, d = pool.shape
    index = pool.get_device()
    kv = cache.packed_kv(hkv, d)
    requests, blocks, block = cache.block_offsets.shape[0] - 1, _slots(cache), cache.block_size
    held = _ints(lengths, (requests,), "lengths", index)
    keep, longest = _kept(keep), cache.max_blocks * block
    if first < 0 or last < 0 or first + last > keep:
        raise ValueError(f"keep = {keep} must hold the first {first} and the last {last} tokens")
    source = _weights(weights, (hkv, blocks, block), "weights", index)
    goal = source if weights_out is None else _weights(weights_out, (hkv, blocks, block), "weights_out", index)
    lo = hi = None
    if cache.lo.shape[1]:
        for name, x in (("lo", cache.lo), ("hi", cache.hi)):
            if x.shape != (hkv, blocks, d) or x.dtype is not torch.float32 or x.get_device() != index or \
                    not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous FP32 [Hkv, blocks, D] on the cache's device")
        lo, hi = cache.lo.data_ptr(), cache.hi.data_ptr()
    if workspace is None:
        need = _evict_bytes(index, L.dtype_code(pool), hkv, block, d, cache.page_size, requests, blocks, keep, longest)
        workspace = weights.new_empty((need,), dtype=torch.uint8)
    else:
        if workspace.get_device() != index or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous and on the cache's device")
        need = workspace.numel()
    kept = lengths.new_empty((requests, hkv, keep))
    now = lengths.new_empty((requests,))
    rc = L.on_device(index, L.load().stk_evict_tokens, kv, pages, requests, blocks, held, keep, first, last, longest,
                     source, goal, lo, hi, kept.data_ptr(), now.data_ptr(), workspace.data_ptr(), need, L.status_ptr(),
                     L.raw_stream(index))
    if rc:
        L.check(rc, "evict")
    return now, kept
