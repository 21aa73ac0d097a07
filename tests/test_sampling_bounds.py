"""Sampling where the thresholds of top_k and top_p meet: in one bin of the
kernel's histogram, among neighbouring numbers, among more tokens than one CTA
sorts, behind masked tokens. Each row is drawn from with many numbers and
compared with the definition in 64 bits; a decision that lies within four times
what the masses' sums may be off by (whole numbers of 2^-44, 2e-14 relative)
from its border is left out."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def definition(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens drawn from the row x by the numbers u, and which of them no rounding decides."""
    x, u = x.double().cpu().numpy(), u.double().cpu().numpy()
    temperature, top_p, min_p = (float(np.float32(y)) for y in (temperature, top_p, min_p))
    best = np.argsort(-x, kind="stable")
    e = np.exp((x - x[best[0]]) / temperature)
    rough = e[(e > 0) & (e < 1)]
    off = 2.0 ** -50 + float((2.0 ** -45 + 2e-14 * rough).sum()) / float(e.sum())
    near = 1.0
    if 0 < top_k < len(x):
        best = best[:top_k]
    if top_p < 1:
        total = math.fsum(e[best])
        before = np.concatenate(([0.0], np.cumsum(e[best], dtype=np.longdouble)))[:-1]
        near = min(near, float(np.abs(before[1:] - top_p * total).min(initial=total)) / total)
        best = best[:max(1, int((before < top_p * total).sum()))]
    if min_p > 0:
        near = min(near, float(np.abs(e[best] - min(min_p, 1.0))[e[best] != 1].min(initial=1.0)))
        best = best[e[best] >= min(min_p, 1.0)]
    best = np.sort(best[e[best] > 0])
    sums = np.cumsum(e[best], dtype=np.longdouble)
    at = u * sums[-1]
    place = np.minimum(np.searchsorted(sums, at, side="right"), len(best) - 1)
    gap = np.minimum(np.abs(sums[place] - at), np.where(place > 0, np.abs(sums[np.maximum(place, 1) - 1] - at), 1.0))
    gap = np.where(place == len(best) - 1, np.where(place > 0, np.abs(sums[np.maximum(place, 1) - 1] - at), 1.0), gap)
    return best[place], np.minimum(near, (gap / sums[-1]).astype(float)) >= 4 * off


def check(x, u, *, least=0.9, **more):
    """Draws from the row x by each number, twice."""
    from strict_topk_overlap_b200 import sampling
    rows = x.expand(u.shape[0], x.shape[-1])
    got = sampling.sample(rows, u, **more)
    assert torch.equal(sampling.sample(rows, u, **more), got), more
    want, sure = definition(x, u, **more)
    assert sure.mean() >= least, (more, sure.mean())
    got = got.cpu().numpy()
    bad = (got != want) & sure
    assert not bad.any(), (more, int(bad.sum()), len(want), np.nonzero(bad)[0][:5], got[bad][:5], want[bad][:5])


def numbers(n, seed=0):
    """Numbers in [0, 1), one in each n-th of it."""
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.arange(n, device=DEV) + 0.98 * torch.rand((n,), generator=g, device=DEV) + 0.01) / n


@gpu
@pytest.mark.parametrize("v", [4000, 30000, 200000])
@pytest.mark.parametrize("top_k", [995, 1000, 1010, 1024])
def test_both_thresholds_in_one_bin(v, top_k):
    """1,050 tokens lie up to the bin in which top_k cuts, and top_p's mass ends in that bin as well."""
    x = torch.full((v,), -40.0)
    place = torch.randperm(v, generator=torch.Generator().manual_seed(top_k))[:1050]
    x[place[:990]] = torch.linspace(0.5, 0.0, 990)
    x[place[990:]] = -0.5 - torch.arange(60) * 1e-4
    for top_p in (0.99, 0.999, 0.9999):
        check(x.to(DEV), numbers(2048), top_k=top_k, top_p=top_p)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [8000, 131072])
@pytest.mark.parametrize("spread", [0.02, 0.5, 2.5])
def test_top_k_with_top_p(dtype, v, spread):
    """Around the 1,024 tokens that one CTA sorts, in rows from nearly flat to steep."""
    g = torch.Generator(DEV).manual_seed(v)
    for i, top_k in enumerate((50, 300, 900, 1000, 1020, 1023, 1024, 1025, 2000)):
        x = (spread * torch.randn((v,), generator=g, device=DEV)).to(dtype)
        for top_p in (0.5, 0.9, 0.99, 0.999):
            check(x, numbers(64, i), least=0.5, temperature=(1.0, 1.3)[i % 2], top_k=top_k, top_p=top_p,
                  min_p=0.01 if i % 3 == 2 else 0.0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_crowded_bins(dtype):
    """Thousands of tokens within one bin, different ones and equal ones, at a small top_k."""
    g = torch.Generator(DEV).manual_seed(1)
    for v in (5000, 70000):
        x = (1 + torch.rand((v,), generator=g, device=DEV) / 100).to(dtype)
        for top_k in (1, 50, 1023, 1025, 3000):
            for top_p in (1.0, 0.999, 0.6):
                check(x, numbers(128), least=0.5, top_k=top_k, top_p=top_p)


@gpu
@pytest.mark.parametrize("more", [dict(top_k=1500), dict(top_k=1100), dict(top_k=1500, top_p=0.97), dict(top_p=0.9), dict(top_p=0.6)])
@pytest.mark.parametrize("v", [4000, 60000])
def test_neighbouring_numbers(v, more):
    """Logits one unit in the last place apart: the first one that does not stay is the next number below the last that does."""
    x = torch.full((v,), -40.0)
    place = torch.randperm(v, generator=torch.Generator().manual_seed(2))[:1800]
    ulp = 2.0 ** -24
    x[place[:900]] = 1.0
    x[place[900:]] = 0.75 - torch.arange(900) * ulp
    check(x.to(DEV), numbers(8192), **more)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("live", [1, 200, 1024, 1500])
def test_masked_vocabularies(dtype, live):
    """Most tokens masked with -inf: fewer than top_k, as many, more."""
    g = torch.Generator(DEV).manual_seed(3)
    for v in (3000, 131072):
        x = torch.full((v,), float("-inf"), device=DEV)
        x[torch.randperm(v, generator=g, device=DEV)[:live]] = 2.5 * torch.randn((live,), generator=g, device=DEV)
        for more in (dict(), dict(top_k=1000), dict(top_k=1000, top_p=0.95), dict(top_p=0.95), dict(top_k=200, min_p=0.05)):
            check(x.to(dtype), numbers(64), least=0.5, **more)
