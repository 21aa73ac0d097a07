"""64-bit restatements of the key weights, of eviction from a paged cache and
of sampling, one request, head or row at a time, from their definitions."""
from __future__ import annotations

import torch


def key_weights(q, k, lse, lo, hi, pos, *, scale, softcap=0.0, slopes=None):
    """One request: q [n, Hq, D], k [Hkv, keys, D], lse [n, Hq]; token i sees keys
    lo[i] <= j < hi[i]. Returns the weights [Hkv, keys] that the keys receive,
    and their sums weighted by (a) the magnitude that the row's score is summed
    from and (b) the magnitudes of score and lse."""
    n, hq, d = q.shape
    hkv, keys = k.shape[0], k.shape[1]
    g = hq // hkv
    j = torch.arange(keys, device=q.device)
    lo, hi, pos = (torch.as_tensor(x, device=q.device)[:, None] for x in (lo, hi, pos))
    x, k = q.double().view(n, hkv, g, d), k.double()
    s = torch.einsum("nhgd,hkd->nhgk", x, k).reshape(n, hq, keys) * scale
    size = torch.einsum("nhgd,hkd->nhgk", x.abs(), k.abs()).reshape(n, hq, keys) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        bias = slopes.double()[:, None] * (pos - j).abs()[:, None]
        s, size = s - bias, size + bias
    lse = lse.double()[..., None]
    seen = ((j >= lo) & (j < hi))[:, None] & (lse != float("-inf"))
    w = torch.where(seen, torch.exp(s - lse), 0.0)
    some = w != 0
    per = lambda y: torch.where(some, w * y, 0.0).view(n, hkv, g, keys).sum((0, 2))  # noqa: E731
    return w.view(n, hkv, g, keys).sum((0, 2)), per(size), per(s.abs() + lse.abs())


def kept_tokens(weights, keep, first, last):
    """Places of the tokens that stay of one row of weights [n], ascending."""
    n = weights.shape[0]
    places = list(range(n))
    if n <= keep:
        return places
    rank = [(float("inf") if w != w else 0.0 + w, w != w) for w in weights.tolist()]
    middle = sorted(places[first:n - last], key=lambda j: (not rank[j][1], -rank[j][0], j))
    return sorted(places[:first] + middle[:keep - first - last] + places[n - last:])


def evict(cache, weights, lengths, keep, first, last):
    """The cache's tensors, the weights, the lengths and the kept places after an eviction, one row at a time."""
    k, v, out = cache.k_pages.clone(), cache.v_pages.clone(), torch.zeros_like(weights)
    lo, hi = cache.lo.clone(), cache.hi.clone()
    hkv, block, page = cache.hkv, cache.block_size, cache.page_size
    flat, flat_out = weights.view(hkv, -1), out.view(hkv, -1)
    off, ppb, d = cache.block_offsets.tolist(), block // page, cache.dim
    kept = torch.full((len(lengths), hkv, keep), -1, dtype=torch.int32, device=k.device)
    for r, n in enumerate(lengths):
        pages = cache.page_table[off[r] * ppb:off[r + 1] * ppb].long()
        for h in range(hkv):
            row = flat[h, off[r] * block:off[r] * block + n]
            stay = torch.tensor(kept_tokens(row, keep, first, last), device=k.device, dtype=torch.long)
            m = stay.numel()
            kept[r, h, :m] = stay.int()
            flat_out[h, off[r] * block:off[r] * block + m] = row[stay]
            if n <= keep:
                continue
            to = torch.arange(m, device=k.device)
            for pool, old in ((k, cache.k_pages), (v, cache.v_pages)):
                pool[pages[to // page], h, to % page] = old[pages[stay // page], h, stay % page]
            for j in range(-(-n // block)):
                at = torch.arange(j * block, max(j * block, min((j + 1) * block, m)), device=k.device)
                if lo.shape[1] == 0 or (at.numel() == block and bool((stay[at] == at).all())):
                    continue
                keys = k[pages[at // page], h, at % page].float() if at.numel() else None
                lo[h, off[r] + j] = torch.full((d,), 1e30, device=k.device) if keys is None else keys.amin(0)
                hi[h, off[r] + j] = torch.full((d,), -1e30, device=k.device) if keys is None else keys.amax(0)
    return k, v, lo, hi, out, [min(n, keep) for n in lengths], kept


def sample(logits, uniform, temperature, top_k, top_p, min_p):
    """One row: the token drawn, how near a decision that masses make came to its
    border, and how far sums of masses may be off that are added as whole
    numbers of 2^-44 (the largest mass is 1), both relative to the whole mass."""
    import math

    import numpy as np
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    v = len(x)
    f = lambda y: float(np.float32(y))  # noqa: E731
    best = np.lexsort((np.arange(v), -x))
    if x[best[0]] == -np.inf:
        return -1, 1.0, 0.0
    if f(temperature) <= 0:
        return int(best[0]), 1.0, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(x == x[best[0]], 1.0, np.exp((x - x[best[0]]) / f(temperature)))
    e = np.where(x == -np.inf, 0.0, e)
    near, rough = 1.0, e[(e > 0) & (e < 1)]  # (a mass of 1 is exact)
    off = 2.0 ** -50 + float((2.0 ** -45 + 2e-14 * rough).sum()) / float(e.sum())
    if 0 < top_k < v:
        best = best[:top_k]
    if f(top_p) < 1:
        before = np.concatenate(([0.0], np.cumsum(e[best], dtype=np.longdouble)))[:-1]
        total = math.fsum(e[best])
        near = min(near, float(np.abs(before[1:] - f(top_p) * total).min(initial=total)) / total)
        best = best[:max(1, int((before < f(top_p) * total).sum()))]
    if f(min_p) > 0:
        near = min(near, float(np.abs(e[best] - min(f(min_p), 1.0))[e[best] != 1].min(initial=1.0)))
        best = best[e[best] >= min(f(min_p), 1.0)]
    best = np.sort(best)
    sums = np.cumsum(e[best], dtype=np.longdouble)
    at = f(uniform) * sums[-1]
    near = min(near, float(np.abs(sums[:-1] - at).min(initial=1.0)) / float(sums[-1]))
    return int(best[min(int(np.searchsorted(sums, at, side="right")), len(best) - 1)]), near, off
