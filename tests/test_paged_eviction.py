"""Key weights and eviction against their definitions in 64 bits.

A key's weight is a sum over rows of w = exp(s - lse). In FP32 the exponent is
off by (D + 16) 2^-24 A for a dot product of D terms, its scaling, cap and bias
(A the magnitude it is summed from), by 4 roundings of 2^-24 (|s| + |lse|) in
powers of two (scale, log-sum-exp and their difference), and the exponential
itself by 2^-21 relative. A capped score is off by 2^-22 of itself more. The
sums are taken in chains of at most 128 additions (56 pairs of rows within a
tile, then tiles, then parts, then what was there before), so they are off by
128 * 2^-24 of the sum. Eviction moves values and is exact."""
from __future__ import annotations

import pytest
import torch

from oracle import eviction as E
from oracle import paged_dense as O
from test_paged_attention import _cache, _ints

gpu = pytest.mark.gpu
DEV = "cuda"
BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32


def _weigh(lengths, new, hq, hkv, d, block, page, dtype, seed, *, mask="causal", softcap=0.0, biased=False, scale=None,
           strided=False, spread=1.0, odd_lse=False, most=None):
    from strict_topk_overlap_b200 import paged_attention, paged_eviction
    cache = _cache(lengths, hkv, d, block, page, dtype, seed)
    g = torch.Generator(DEV).manual_seed(seed + 1)
    t = sum(new)
    q = (spread * torch.randn((t, hq + (3 if strided else 0), d + (8 if strided else 0)), generator=g, device=DEV)).to(dtype)
    if strided:
        q = q[:, 1:hq + 1, :d]
    pos = [p for n, length in zip(new, lengths) for p in range(length - n, length)]
    lo, hi = [0] * t, [p + 1 for p in pos]
    if mask == "window":
        lo = [max(0, p - 36) for p in pos]
    elif mask == "documents":
        lo = [p // 29 * 29 for p in pos]
    elif mask == "prefix":
        hi = [max(p + 1, 75) for p in pos]
    elif mask == "odd":  # empty intervals, ends beyond the cache, negative starts, single keys
        lo = [(-4, 7, p, 30, p + 1)[i % 5] for i, p in enumerate(pos)]
        hi = [(1 << 30, 7, p + 1, 20, p + 1)[i % 5] for i, p in enumerate(pos)]
    offsets = _ints([0] + list(torch.tensor(new).cumsum(0))) if any(n != 1 for n in new) else None
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if biased else None
    args = dict(token_offsets=offsets, max_tokens=most or max(new), softcap=softcap, slopes=slopes, scale=scale,
                kv_lo=_ints(lo) if mask in ("window", "documents", "odd") else None,
                kv_hi=_ints(hi) if mask in ("prefix", "odd") else None)
    _, lse = paged_attention.attention(q, cache, _ints(lengths), return_lse=True, **args)
    if odd_lse:
        lse[::3] = float("-inf")
    weights = paged_eviction.empty_weights(cache)
    weights.copy_(0.01 * torch.rand(weights.shape, generator=g, device=DEV))
    before = weights.clone()
    got = paged_eviction.accumulate_weights(weights, q, cache, _ints(lengths), lse, **args)
    assert got is weights
    off, start = cache.block_offsets.tolist(), 0
    want, tol = before.double().view(hkv, -1), torch.zeros_like(before, dtype=torch.float64).view(hkv, -1)
    for r, (n, length) in enumerate(zip(new, lengths)):
        if n == 0:
            continue
        rows = slice(start, start + n)
        k = O.gather(cache.k_pages, cache.page_table, off, block, page, r, length)
        w, by_size, by_score = E.key_weights(q[rows], k, lse[rows], lo[rows], hi[rows], pos[start:start + n],
                                             scale=scale or d ** -0.5, softcap=softcap, slopes=slopes)
        at = slice(off[r] * block, off[r] * block + length)
        want[:, at] += w
        tol[:, at] = (d + 16) * 2.0 ** -24 * by_size + (8 if softcap else 4) * 2.0 ** -24 * by_score + 2.0 ** -21 * w
        tol[:, at] += 128 * 2.0 ** -24 * want[:, at].abs()
        start += n
    off_by = (got.view(hkv, -1).double() - want).abs()
    bad = ~(off_by <= tol)  # slots without a key that is seen are left bit for bit
    assert not bool(bad.any()), (bad.nonzero()[:5].tolist(), off_by[bad][:5], tol[bad][:5], want[bad][:5])


@gpu
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("lengths,new", [
    ([1], [1]), ([40, 1, 300], [1, 1, 1]), ([5, 129, 513], [3, 1, 7]), ([257, 64], [100, 64]), ([700], [700]),
    ([300, 31, 1000, 0], [300, 0, 129, 0])])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 2, 64), (12, 1, 128)])
def test_weights(lengths, new, hq, hkv, d, dtype):
    _weigh(lengths, new, hq, hkv, d, 32, 16, dtype, 3)


@gpu
@pytest.mark.parametrize("mask", ["window", "documents", "prefix", "odd"])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HALF, 64), (F32, 128)])
@pytest.mark.parametrize("lengths,new", [([90, 600, 33], [1, 1, 1]), ([300, 700], [300, 211])])
def test_weights_of_masks(mask, dtype, d, lengths, new):
    _weigh(lengths, new, 8, 2, d, 32, 16, dtype, 4, mask=mask)


@gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HALF, 64), (F32, 96)])
@pytest.mark.parametrize("more", [
    dict(softcap=50.0), dict(softcap=2.0, spread=3.0), dict(softcap=8.0, spread=3.0), dict(biased=True),
    dict(biased=True, softcap=30.0, mask="window"), dict(scale=0.25), dict(strided=True), dict(odd_lse=True)])
@pytest.mark.parametrize("lengths,new", [([200, 45], [1, 1]), ([400, 290], [400, 20])])
def test_weights_of_scores(dtype, d, more, lengths, new):
    _weigh(lengths, new, 8, 2, d, 32, 16, dtype, 5, **more)


@gpu
@pytest.mark.parametrize("hq,hkv,d,block,page,dtype", [
    (32, 32, 128, 32, 32, BF), (7, 1, 64, 64, 8, HALF), (130, 1, 128, 128, 128, BF), (96, 1, 64, 256, 256, HALF), (57, 1, 64, 32, 16, BF),
    (4, 2, 72, 32, 16, BF), (4, 4, 256, 32, 8, HALF), (2, 1, 80, 30, 10, F32), (6, 3, 33, 12, 4, F32), (1, 1, 1, 4, 4, F32),
    (2, 2, 1024, 16, 16, F32)])
@pytest.mark.parametrize("lengths,new", [([30, 260], [1, 1]), ([150, 300], [150, 20])])
def test_weights_of_layouts(hq, hkv, d, block, page, dtype, lengths, new):
    _weigh(lengths, new, hq, hkv, d, block, page, dtype, 6)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_weights_of_many_requests(dtype):
    """More requests than one window of the walk, some without new tokens."""
    lengths = [(37 * r) % 411 + 1 for r in range(77)]
    _weigh(lengths, [1] * 77, 8, 2, 128, 32, 16, dtype, 7)
    _weigh(lengths, [min(n, (r * 5) % 13) for r, n in enumerate(lengths)], 8, 2, 128, 32, 16, dtype, 8, mask="window")


@gpu
def test_weights_in_parts():
    """Rows in parts whose sums are joined: the same bits whenever it runs, and within the bounds."""
    _weigh([3001], [3001], 8, 2, 128, 32, 16, BF, 9)
    _weigh([2000, 3], [1500, 3], 4, 1, 64, 32, 16, HALF, 10, mask="documents")


def _filled(lengths, hkv, d, block, page, dtype, seed, *, room=0, bounds=True):
    """A pool with slots that no token fills, its bounds those of the tokens (1e30 where a block has none)."""
    from strict_topk_overlap_b200 import paged
    cache = _cache(lengths, hkv, d, block, page, dtype, seed, room=room)
    if not bounds:
        return cache
    off, ppb, total = cache.block_offsets.tolist(), block // page, cache.block_offsets[-1].item()
    lo, hi = torch.full((hkv, total, d), 1e30, device=DEV), torch.full((hkv, total, d), -1e30, device=DEV)
    for r, n in enumerate(lengths):
        k = O.gather(cache.k_pages, cache.page_table, off, block, page, r, n).float()
        for j in range(-(-n // block)):
            lo[:, off[r] + j], hi[:, off[r] + j] = k[:, j * block:(j + 1) * block].amin(1), k[:, j * block:(j + 1) * block].amax(1)
    return paged.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table, cache.block_offsets, lo, hi, block, page,
                              cache.max_blocks)


def _same(got, want):
    return torch.equal(got.view(torch.uint8) if got.is_floating_point() else got,
                       want.view(torch.uint8) if want.is_floating_point() else want)


def _evict(lengths, keep, hkv, d, block, page, dtype, seed, *, first=0, last=0, kind="random", in_place=False, room=0, bounds=True):
    from strict_topk_overlap_b200 import paged_eviction
    cache = _filled(lengths, hkv, d, block, page, dtype, seed, room=room, bounds=bounds)
    g = torch.Generator(DEV).manual_seed(seed + 1)
    weights = paged_eviction.empty_weights(cache)
    x = torch.exp(2 * torch.randn(weights.shape, generator=g, device=DEV))
    if kind == "ties":
        x = (4 * torch.rand(weights.shape, generator=g, device=DEV)).floor()
    elif kind == "equal":
        x = torch.zeros_like(x)
    elif kind == "signs":  # negative ones, zeros of either sign, infinities and NaN
        x = torch.randn(weights.shape, generator=g, device=DEV)
        pick = torch.randint(0, 9, weights.shape, generator=g, device=DEV)
        for i, value in enumerate((0.0, -0.0, float("inf"), float("-inf"), float("nan"))):
            x[pick == i] = value
    elif kind == "rising":
        x = torch.arange(x.numel(), device=DEV).float().view(x.shape)
    elif kind == "falling":
        x = -torch.arange(x.numel(), device=DEV).float().view(x.shape)
    weights.copy_(x)
    want = E.evict(cache, weights, lengths, keep, first, last)
    out = None if in_place else torch.full_like(weights, 7.0)
    now, kept = paged_eviction.evict(cache, weights, _ints(lengths), keep, first=first, last=last, weights_out=out)
    got = (cache.k_pages, cache.v_pages, cache.lo, cache.hi, weights if in_place else out, now, kept)
    names = ("k", "v", "lo", "hi", "weights", "lengths", "kept")
    want = (*want[:5], _ints(want[5]), want[6])
    if not in_place:
        assert _same(weights, x)
    off = cache.block_offsets.tolist()
    for name, a, b in zip(reversed(names), reversed(got), reversed(want)):
        if name == "weights":  # slots of no request's blocks are nobody's
            a, b = a[:, :off[-1]], b[:, :off[-1]]
        assert _same(a, b), (name, (a != b).nonzero()[:8].tolist())
    return cache, now, kept


@gpu
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "signs", "rising", "falling"])
@pytest.mark.parametrize("lengths,keep,first,last", [
    ([100], 40, 0, 0), ([300, 20, 64, 1], 64, 4, 16), ([513, 700], 512, 0, 1), ([90, 200], 1, 0, 0), ([90, 200], 32, 16, 16),
    ([33, 1000], 999, 3, 0), ([4100], 300, 10, 50), ([5, 0, 40], 8, 1, 1)])
def test_evict(kind, lengths, keep, first, last):
    _evict(lengths, keep, 2, 128, 32, 16, BF, 20, first=first, last=last, kind=kind)
    _evict(lengths, keep, 3, 64, 64, 32, HALF, 21, first=first, last=last, kind=kind, in_place=True, room=100)


@gpu
@pytest.mark.parametrize("hkv,d,block,page,dtype", [
    (8, 128, 32, 16, F32), (1, 256, 128, 128, BF), (2, 96, 24, 8, BF), (3, 40, 6, 3, HALF), (2, 33, 12, 4, F32), (2, 33, 7, 7, HALF),
    (1, 1, 4, 4, BF), (2, 1024, 16, 16, F32), (2, 520, 32, 16, HALF), (16, 64, 256, 16, BF)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_layouts(hkv, d, block, page, dtype, in_place):
    _evict([200, 77], 60, hkv, d, block, page, dtype, 22, first=2, last=5, in_place=in_place)
    _evict([200, 77], 70, hkv, d, block, page, dtype, 23, kind="rising", in_place=in_place, bounds=False)


@gpu
def test_evict_long():
    """Rows that clusters of several CTAs share, and chunks that wait for earlier ones across the whole grid."""
    _evict([50000], 30000, 2, 64, 32, 16, BF, 24, first=64, last=500)
    _evict([20000, 9000, 16385], 16384, 1, 64, 64, 16, HALF, 25, kind="ties")
    _evict([120000], 119000, 1, 64, 32, 16, BF, 26, in_place=True)


@gpu
def test_evict_again():
    """Evicting what an eviction left: nothing at the same number, and the first part of the first selection below it."""
    cache, now, kept = _evict([400, 90], 128, 2, 64, 32, 16, BF, 27, last=4)
    from strict_topk_overlap_b200 import paged_eviction
    k, lo = cache.k_pages.clone(), cache.lo.clone()
    w = paged_eviction.empty_weights(cache)
    now2, kept2 = paged_eviction.evict(cache, w, now, 128)
    assert torch.equal(now2, now) and _same(cache.k_pages, k) and _same(cache.lo, lo)
    assert kept2[0, 0].tolist() == list(range(128)) and kept2[1, 1].tolist() == list(range(90)) + [-1] * 38
