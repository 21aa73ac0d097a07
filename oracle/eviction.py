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
