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
