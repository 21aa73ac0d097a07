"""64-bit restatements of the paged token append and the dense paged attention,
one request and one token at a time, from their definitions."""
from __future__ import annotations

import torch


def gather(pool, table, block_offsets, block, page, r, count):
    """The first ``count`` tokens of request r: [Hkv, count, D] of a pool [pages, Hkv, page, D]."""
    ppb = block // page
    pages = table[block_offsets[r] * ppb:block_offsets[r + 1] * ppb].long()
    return pool[pages].transpose(0, 1).flatten(1, 2)[:, :count]


def rotate(x, cos, sin, interleaved, angles):
    """x [T, H, D] with pair p turned by the angle of table row angles[t, p], in 64 bits."""
    x = x.double()
    pairs = cos.shape[1]
    c = cos.double().gather(0, angles)[:, None]
    s = sin.double().gather(0, angles)[:, None]
    i = torch.arange(pairs, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    out = x.clone()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def attention(q, k, v, lo, hi, pos, *, scale, softcap=0.0, slopes=None):
    """One request: q [n, Hq, D], k and v [Hkv, keys, D]; token i sees keys
    lo[i] <= j < hi[i]. Returns out [n, Hq, D], lse [n, Hq] and, per row, the
    largest magnitude that a score of noticeable weight is summed from and the
    largest finite value of its head. Unseen keys take no part, whatever they hold."""
    n, hq, d = q.shape
    hkv, keys = k.shape[0], k.shape[1]
    g = hq // hkv
    j = torch.arange(keys, device=q.device)
    lo, hi, pos = (torch.as_tensor(x, device=q.device)[:, None] for x in (lo, hi, pos))
    seen = ((j >= lo) & (j < hi))[:, None]  # [n, 1, keys]
    x = q.double().view(n, hkv, g, d)
    k, v = k.double(), v.double()
    s = torch.einsum("nhgd,hkd->nhgk", x, k).reshape(n, hq, keys) * scale
    size = torch.einsum("nhgd,hkd->nhgk", x.abs(), k.abs()).reshape(n, hq, keys) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        bias = slopes.double()[:, None] * (pos - j).abs()[:, None]
        s, size = s - bias, size + bias
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = w.sum(-1, keepdim=True)
    share = torch.where(total == 0, 0.0, w / total).view(n, hkv, g, keys)
    finite = v.isfinite()
    out = torch.einsum("nhgk,hkd->nhgd", share, torch.where(finite, v, 0.0))
    for t in (~finite).any(-1).any(0).nonzero().flatten().tolist():
        rows = seen[:, 0, t].nonzero().flatten()
        part = torch.where(finite[:, t], 0.0, v[:, t])[None, :, None]
        out[rows] += share[rows][..., t, None] * part
    size = torch.where(w > 2.0 ** -30, size, 0.0).amax(-1)
    vmax = torch.where(finite, v.abs(), 0.0).amax((1, 2)).repeat_interleave(g).expand(n, hq)
    return out.reshape(n, hq, d), (top + torch.log(total)).squeeze(-1), size, vmax
