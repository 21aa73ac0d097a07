"""Filling a paged cache: prompts, pieces of prompts and single tokens.

``empty_paged_cache`` allocates a page pool with its table; ``append_tokens``
(stk_append_tokens) rotates new keys and queries by their positions, writes
keys and values into their pages and keeps the blocks' key bounds current, in
one launch. What it leaves is what ``paged.select_blocks`` and the attention
calls read. New: the reference starts from a filled dense cache.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from .paged import PagedKVCache
from .rotary import Rotary


def empty_paged_cache(capacities, hkv, dim, block_size, page_size, *, dtype=torch.bfloat16, bounds=True,
                      generator=None, device="cuda") -> PagedKVCache:
    """A pool for requests of up to ``capacities`` tokens, its pages handed out
    in a seeded random order. ``bounds=False`` keeps no per-block key bounds
    (a cache that no block selection reads). The pool is zeroed; a block
    without tokens has bounds that no query scores high: lo = 3e38, hi = -3e38."""
    if not capacities or min(capacities) <= 0:
        raise ValueError("every request needs room for at least one token")
    if block_size % page_size:
        raise ValueError(f"page size {page_size} must divide the block size {block_size}")
    blocks = [-(-int(c) // block_size) for c in capacities]
    total = sum(blocks)
    pages = total * (block_size // page_size)
    offsets = [0]
    for n in blocks:
        offsets.append(offsets[-1] + n)
    table = torch.randperm(pages, generator=generator).to(torch.int32).to(device)
    k = torch.zeros((pages, hkv, page_size, dim), dtype=dtype, device=device)
    lo = torch.full((hkv, total if bounds else 0, dim), 3e38, device=device)
    return PagedKVCache(k, torch.zeros_like(k), table, torch.tensor(offsets, dtype=torch.int32, device=device), lo,
                        -lo, block_size, page_size, max(blocks))


def _check_ints(t, shape, name, device):
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be contiguous int32 of shape {tuple(shape)} on the cache's device")


def _check_rows(x, cache, heads, name):
    if x.ndim != 3 or x.shape[1] != heads or x.shape[2] != cache.k_pages.shape[3]:
        raise ValueError(f"{name} must be [T, {heads}, D]")
    if x.dtype != cache.k_pages.dtype or x.device != cache.k_pages.device:
        raise ValueError(f"{name} must have the cache's dtype and device")
    if x.stride(2) != 1 and x.shape[2] > 1:
        raise ValueError(f"{name} must have unit stride along D")


def append_tokens(cache: PagedKVCache, k, v, lengths, *, token_offsets=None, q=None, rotary: Rotary | None = None,
                  positions=None, q_out=None):
    """Append packed new tokens' k, v [T, Hkv, D] to the cache: request r's
    tokens token_offsets[r] .. token_offsets[r + 1] (int32 [R + 1]; None: one
    token per request) become its tokens lengths[r] (int32 [R], before the
    call), lengths[r] + 1, ... With ``rotary``, k and q [T, Hq, D] are rotated
    by ``positions`` (int32 [T], or [axes, T]; None: the token's place). k, v
    and q may be slices of one projection's output (any token and head
    strides). Updates the pages and, where the cache keeps them, the blocks'
    lo / hi; returns the rotated q [T, Hq, D] (``q_out``, which may be q
    itself), or None without q."""
    pool, hkv = cache.k_pages, cache.hkv
    dev, requests = pool.device, cache.requests
    _check_rows(k, cache, hkv, "k")
    _check_rows(v, cache, hkv, "v")
    t = k.shape[0]
    if v.shape[0] != t:
        raise ValueError("k and v must have the same number of tokens")
    _check_ints(lengths, (requests,), "lengths", dev)
    if token_offsets is not None:
        _check_ints(token_offsets, (requests + 1,), "token_offsets", dev)
    elif t != requests:
        raise ValueError("without token_offsets there must be one token per request")
    hq = qt = qh = 0
    if q is not None:
        hq = q.shape[1] if q.ndim == 3 else 0
        _check_rows(q, cache, hq, "q")
        if q.shape[0] != t or hq == 0 or hq % hkv:
            raise ValueError("q must be [T, Hq, D] with Hq a multiple of the KV heads")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.device != dev or not q_out.is_contiguous():
            raise ValueError("q_out must be contiguous, of q's shape, dtype and device")
        qt, qh = q.stride(0), q.stride(1)
    turn = None
    if rotary is not None:
        cos, sin, axis = rotary.cos, rotary.sin, rotary.axis
        if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or \
                cos.device != dev or sin.device != dev or not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("rotary cos / sin must be contiguous FP32 [positions, pairs] on the cache's device")
        axes = 1
        if positions is not None:
            axes = positions.shape[0] if positions.ndim == 2 else 1
            _check_ints(positions, (axes, t) if positions.ndim == 2 else (t,), "positions", dev)
        if axis is not None:
            if axis.dtype != torch.uint8 or axis.shape != cos.shape[1:] or axis.device != dev or \
                    not axis.is_contiguous():
                raise ValueError("rotary axis must be uint8 [pairs] on the cache's device")
            if positions is None:
                raise ValueError("several rotary axes need positions [axes, T]")
        elif axes > 1:
            raise ValueError("positions with several axes need a rotary axis for each pair")
        turn = L.StkRotary(cos.data_ptr(), sin.data_ptr(), cos.shape[1], cos.shape[0], int(rotary.interleaved), axes,
                           L.ptr(axis))
    elif positions is not None:
        raise ValueError("positions need a rotary table")
    bounds = cache.total_blocks > 0
    kv = cache.kv()
    rc = L.load().stk_append_tokens(
        kv, pool.shape[0], requests, cache.total_blocks if bounds else 1, t, k.data_ptr(), k.stride(0), k.stride(1),
        v.data_ptr(), v.stride(0), v.stride(1), L.ptr(q), qt, qh, hq, L.ptr(q_out) if q is not None else None,
        lengths.data_ptr(), L.ptr(token_offsets), L.ptr(positions), turn, cache.lo.data_ptr() if bounds else None,
        cache.hi.data_ptr() if bounds else None, L.status_ptr(), L.stream_of(pool))
    L.check(rc, "append_tokens")
    return q_out if q is not None else None
