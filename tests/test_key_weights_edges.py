"""Key weights at single infinite elements of keys and in long sums, and what the
calls return and report."""
from __future__ import annotations

import pytest
import torch

from oracle import eviction as E
from oracle import paged_dense as O
from test_paged_attention import _cache, _ints

gpu = pytest.mark.gpu
DEV = "cuda"
BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def status():
    from strict_topk_overlap_b200 import _lib as L
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    L.set_status_tensor(word)
    yield word
    L.set_status_tensor(None)


@gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HALF, 64), (F32, 128), (F32, 96)])
@pytest.mark.parametrize("hq", [2, 8, 14, 32])
@pytest.mark.parametrize("new", [1, 3, 30, 200])
@pytest.mark.parametrize("more", [dict(), dict(softcap=20.0), dict(slopes=True), dict(softcap=20.0, slopes=True)])
def test_one_infinite_element(dtype, d, hq, new, more):
    """A key with one infinite element weighs nothing where all scores are -inf, infinitely much where some are +inf, and what
    the cap says where there is one. Bounds as in test_paged_eviction.py; an infinite score is capped without an error."""
    from strict_topk_overlap_b200 import paged_eviction
    hkv, n = 2, 400
    cache = _cache([n], hkv, d, 32, 16, dtype, 5)
    g = torch.Generator(DEV).manual_seed(6)
    q = torch.randn((new, hq, d), generator=g, device=DEV)
    q[..., 0] = -q[..., 0].abs() - 0.1  # all below zero, all above, some of either sign
    q[..., 1] = q[..., 1].abs() + 0.1
    q[..., 2] = torch.where(q[..., 2] == 0, 1.0, q[..., 2])
    q = q.to(dtype)
    infinite = {5: (0, 1.0), 40: (1, 1.0), 77: (2, 1.0), 100: (2, -1.0), 130: (1, -1.0), 190: (0, -1.0)}
    for key, (dim, sign) in infinite.items():
        cache.k_pages[cache.page_table[key // 16].long(), :, key % 16, dim] = sign * float("inf")
    lse = 5 + torch.rand((new, hq), generator=g, device=DEV)
    args = dict(softcap=more.get("softcap", 0.0),
                slopes=torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if more.get("slopes") else None)
    offsets = dict(token_offsets=_ints([0, new]), max_tokens=new) if new > 1 else {}
    got = paged_eviction.accumulate_weights(paged_eviction.empty_weights(cache), q, cache, _ints([n]), lse, **args, **offsets)
    k = O.gather(cache.k_pages, cache.page_table, cache.block_offsets.tolist(), 32, 16, 0, n)
    pos = list(range(n - new, n))
    want, by_size, by_score = E.key_weights(q, k, lse, [0] * new, [p + 1 for p in pos], pos, scale=d ** -0.5, **args)
    got = got.view(hkv, -1)[:, :n].double()
    keys = list(infinite)
    assert torch.equal(got.isnan(), want.isnan()) and not bool(want.isnan().any())
    assert torch.equal(got.isinf(), want.isinf())
    if args["softcap"]:
        by_size[:, keys] = 0
        assert bool((want[:, keys] > 0).all())
    else:
        assert bool((got[:, [5, 130]] == 0).all()) and bool(got[:, [40, 190]].isinf().all())
    live = want.isfinite() & (want != 0)
    tol = (d + 16) * 2.0 ** -24 * by_size + (8 if args["softcap"] else 4) * 2.0 ** -24 * by_score + (2.0 ** -21 + 128 * 2.0 ** -24) * want
    off_by = (got - want).abs()
    assert bool((off_by <= tol)[live].all()), (off_by / want)[live].max()
    assert torch.equal(got == 0, want == 0)


@gpu
def test_errors_are_returned():
    """A call that CUDA refuses (here: a pool of more rows than a tensor map takes) is not run by another kernel instead."""
    from strict_topk_overlap_b200 import _lib as L
    cache = _cache([100], 4, 64, 32, 16, BF, 3)
    kv = cache.packed_kv(4, 64)
    q = torch.randn((1, 8, 64), device=DEV).to(BF)
    lse, weights = torch.zeros((1, 8), device=DEV), torch.zeros((4, 4, 32), device=DEV)
    lengths, lib = _ints([100]), L.load()

    def call(pages):
        return lib.stk_accumulate_weights(kv, pages, q.data_ptr(), 512, 64, 1, 1, 8, 4, lengths.data_ptr(), None, 1, 128, None,
                                          lse.data_ptr(), weights.data_ptr(), None, 0, None, L.raw_stream(0))

    assert call(2 ** 31 - 1) != 0  # (the table names pages of the real pool)
    assert lib.stk_last_error() and not bool(weights.any())
    assert call(cache.k_pages.shape[0]) == 0 and bool(weights.any())


@gpu
def test_queries_that_no_tensor_map_takes():
    """Tokens further apart than a tensor map's strides: the same weights by the other kernel."""
    from strict_topk_overlap_b200 import paged_eviction
    cache = _cache([100], 2, 64, 32, 16, BF, 4)
    q = torch.randn((1, 8, 64), generator=torch.Generator(DEV).manual_seed(2), device=DEV).to(BF)
    lse = torch.full((1, 8), 4.0, device=DEV)
    weigh = lambda x: paged_eviction.accumulate_weights(paged_eviction.empty_weights(cache), x, cache, _ints([100]), lse)  # noqa: E731
    want, got = weigh(q), weigh(q.as_strided((1, 8, 64), (2 ** 40, 64, 1)))
    assert bool(want.any()) and bool(((got - want).abs() <= 1e-5 * want).all())


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_the_first_page_behind_the_pool(status, dtype, new):
    """A table entry that equals the number of pages is outside the pool like any other."""
    from strict_topk_overlap_b200 import paged_eviction
    cache = _cache([100, 70], 2, 128, 32, 16, dtype, 2)
    q = torch.randn((2 * new, 8, 128), generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(dtype)
    lse = torch.full((2 * new, 8), 8.0, device=DEV)
    more = dict(token_offsets=_ints([0, new, 2 * new]), max_tokens=new) if new > 1 else {}

    def weigh():
        return paged_eviction.accumulate_weights(paged_eviction.empty_weights(cache), q, cache, _ints([100, 70]), lse, **more)

    good = weigh()
    assert status.item() == 0
    cache.page_table[1] = cache.k_pages.shape[0]
    got = weigh()
    assert status.item() == 2
    assert torch.equal(got[:, 4:], good[:, 4:]) and torch.equal(got[:, 0, :16], good[:, 0, :16])


@gpu
@pytest.mark.parametrize("hq,hkv,d", [(12, 1, 64), (4, 2, 72)])
def test_long_sums(hq, hkv, d):
    """Thousands of rows on the FP32 units: sums of 64 rows of a warp, then in FP64. Rows that all weigh 0.1 are what a single
    FP32 sum is worst at: its roundings all go the same way."""
    from strict_topk_overlap_b200 import paged_eviction
    n = 4100
    cache = _cache([n], hkv, d, 32, 16, F32, 7)
    q = torch.zeros((n, hq, d), device=DEV)
    lse = torch.full((n, hq), 2.302585, device=DEV)
    got = paged_eviction.accumulate_weights(paged_eviction.empty_weights(cache), q, cache, _ints([n]), lse,
                                            token_offsets=_ints([0, n]), max_tokens=n).view(hkv, -1)[:, :n].double()
    want = (hq // hkv) * torch.arange(n, 0, -1, device=DEV).double() * torch.exp(-lse[0, 0].double())
    # 4 roundings of |s| + |lse|, the exponential, 64 additions of a run, and 4 roundings of what the warps' sums become.
    tol = (4 * 2.302585 * 2.0 ** -24 + 2.0 ** -21 + 68 * 2.0 ** -24) * want
    assert bool(((got - want).abs() <= tol).all()), ((got - want).abs() / want).max()
