"""Filling a paged cache: prompts, pieces of prompts and single tokens.

``empty_paged_cache`` allocates a page pool with its table; ``append_tokens``
(stk_append_tokens) rotates new keys and queries by their positions, writes
keys and values into their pages and keeps the blocks' key bounds current, in
one launch. What it leaves is what ``paged.select_blocks`` and the attention
calls read. The block-sparse calls (``paged.select_blocks``, ``paged.exact``
and the speculative ones) know blocks, not token counts: they attend a
request's last block as a full one, so what they read has to end on a block's
border. ``paged_attention`` knows the lengths and reads any. New: the reference
starts from a filled dense cache.
"""
from __future__ import annotations

import torch

from . import _lib as L
from .paged import PagedKVCache
from .rotary import Rotary


_FLOAT = torch.float32
_NOTHING = 1e30  # lo, and minus hi, of a block without tokens


def empty_paged_cache(capacities, hkv, dim, block_size, page_size, *, dtype=torch.bfloat16, bounds=True,
                      generator=None, device="cuda") -> PagedKVCache:
    """A pool for requests of up to ``capacities`` tokens, its pages handed out
    in a seeded random order. ``bounds=False`` keeps no per-block key bounds
    (a cache that no block selection reads). The pool is zeroed; a block
    without tokens has bounds that no query scores high, lo = 1e30 and
    hi = -1e30: far below every block of tokens, yet with sums over a head that
    FP32 holds, so that selection need not rescore them."""
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
    lo = torch.full((hkv, total if bounds else 0, dim), _NOTHING, device=device)
    return PagedKVCache(k, torch.zeros_like(k), table, torch.tensor(offsets, dtype=torch.int32, device=device), lo,
                        -lo, block_size, page_size, max(blocks))


def _ints(x, shape, name, index):
    """Address of an int32 tensor of this shape on device ``index``."""
    if x.dtype is not torch.int32 or x.shape != shape or x.get_device() != index or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 of shape {shape} on the cache's device")
    return x.data_ptr()


def _rows(x, shape, name, dtype, index):
    """Address and token and head strides of rows [T, heads, D]."""
    if x.shape != shape:
        raise ValueError(f"{name} must be [T, heads, D] = {shape}, got {tuple(x.shape)}")
    if x.dtype is not dtype or x.get_device() != index:
        raise ValueError(f"{name} must have the cache's dtype and device")
    token, head, unit = x.stride()
    if unit != 1 and shape[2] > 1:
        raise ValueError(f"{name} must have unit stride along D")
    return x.data_ptr(), token, head


def _heads(q, hkv):
    """Tokens and heads of q [T, Hq, D]."""
    shape = q.shape
    if len(shape) != 3 or shape[1] == 0 or shape[1] % hkv:
        raise ValueError("q must be [T, Hq, D] with Hq a multiple of the KV heads")
    return shape[0], shape[1]


def _tokens(token_offsets, t, requests, index):
    """Address of the packed tokens' offsets, or None for one token per request."""
    if token_offsets is not None:
        return _ints(token_offsets, (requests + 1,), "token_offsets", index)
    if t != requests:
        raise ValueError("without token_offsets there must be one token per request")
    return None


def _rotary(rotary, positions, t, index):
    """The call's packed stk_rotary and the positions' address."""
    if rotary is None:
        if positions is not None:
            raise ValueError("positions need a rotary table")
        return None, None
    cos, sin, axis = rotary.cos, rotary.sin, rotary.axis
    size = cos.shape
    if len(size) != 2 or sin.shape != size or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or \
            cos.get_device() != index or sin.get_device() != index or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("rotary cos / sin must be contiguous FP32 [positions, pairs] on the cache's device")
    axes, at = 1, None
    if positions is not None:
        axes = positions.shape[0] if positions.ndim == 2 else 1
        at = _ints(positions, (axes, t) if positions.ndim == 2 else (t,), "positions", index)
    if axis is None:
        if axes > 1:
            raise ValueError("positions with several axes need a rotary axis for each pair")
        axis_at = 0
    else:
        if axis.dtype is not torch.uint8 or axis.shape != size[1:] or axis.get_device() != index or \
                not axis.is_contiguous():
            raise ValueError("rotary axis must be uint8 [pairs] on the cache's device")
        if positions is None:
            raise ValueError("several rotary axes need positions [axes, T]")
        axis_at = axis.data_ptr()
    return L.PACK_ROTARY(cos.data_ptr(), sin.data_ptr(), size[1], size[0], rotary.interleaved, axes, axis_at), at


def append_tokens(cache: PagedKVCache, k, v, lengths, *, token_offsets=None, q=None, rotary: Rotary | None = None,
                  positions=None, q_out=None):
    """Append packed new tokens' k, v [T, Hkv, D] to the cache: request r's
    tokens token_offsets[r] .. token_offsets[r + 1] (int32 [R + 1]; None: one
    token per request) become its tokens lengths[r] (int32 [R], before the
    call), lengths[r] + 1, ... With ``rotary``, k and q [T, Hq, D] are rotated
    by ``positions`` (int32 [T], or [axes, T]; None: the token's place). k, v
    and q may be slices of one projection's output (any token and head
    strides). Updates the pages and, where the cache keeps them, the blocks'
    lo / hi (tokens from token_offsets[R] on are padding and stored nowhere);
    returns the rotated q [T, Hq, D] (``q_out``, which may be q
    itself), or None without q."""
    pool = cache.k_pages
    pages, hkv, _, d = pool.shape
    dtype, index = pool.dtype, pool.get_device()
    kv = cache.packed_kv(hkv, d)
    bounds = cache.lo.shape
    requests, blocks = cache.block_offsets.shape[0] - 1, bounds[1]
    t = k.shape[0]
    kp, kt, kh = _rows(k, (t, hkv, d), "k", dtype, index)
    vp, vt, vh = _rows(v, (t, hkv, d), "v", dtype, index)
    before = _ints(lengths, (requests,), "lengths", index)
    offsets = _tokens(token_offsets, t, requests, index)
    qp = qt = qh = hq = out = 0
    if q is not None:
        hq = _heads(q, hkv)[1]
        qp, qt, qh = _rows(q, (t, hq, d), "q", dtype, index)
        if q_out is None:
            q_out = q.new_empty((t, hq, d))
        elif q_out.shape != (t, hq, d) or q_out.dtype is not dtype or q_out.get_device() != index or \
                not q_out.is_contiguous():
            raise ValueError("q_out must be contiguous, of q's shape, dtype and device")
        out = q_out.data_ptr()
    turn, at = _rotary(rotary, positions, t, index)
    lo = hi = None
    if blocks:
        low, high = cache.lo, cache.hi
        if bounds != (hkv, blocks, d) or high.shape != bounds or low.dtype is not _FLOAT or high.dtype is not _FLOAT or \
                low.get_device() != index or high.get_device() != index or not low.is_contiguous() or \
                not high.is_contiguous():
            raise ValueError("lo and hi must be contiguous FP32 [Hkv, blocks, D] on the cache's device")
        lo, hi = low.data_ptr(), high.data_ptr()
    rc = L.on_device(index, L.load().stk_append_tokens, kv, pages, requests, blocks or 1, t, kp, kt, kh, vp, vt, vh, qp,
                     qt, qh, hq, out, before, offsets, at, turn, lo, hi, L.status_ptr(), L.raw_stream(index))
    if rc:
        L.check(rc, "append_tokens")
    return q_out if q is not None else None
