"""Key weights, eviction and sampling at the edges of what they are given: keys
that no token sees, tables and lengths that are wrong, padding, graphs, streams,
addresses off a 16-byte boundary."""
from __future__ import annotations

import pytest
import torch

from oracle import eviction as E
from test_paged_attention import _cache, _ints
from test_paged_eviction import _filled, _same

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


def _weighed(cache, q, lengths, weights=None, lse=None, **more):
    from strict_topk_overlap_b200 import paged_attention, paged_eviction
    if lse is None:
        _, lse = paged_attention.attention(q, cache, lengths, return_lse=True, **more)
    weights = paged_eviction.empty_weights(cache) if weights is None else weights
    return paged_eviction.accumulate_weights(weights, q, cache, lengths, lse, **more), lse


def _queries(t, hq, d, dtype, seed=1):
    return torch.randn((t, hq, d), generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_nobody_sees(status, dtype, new):
    """Behind a sliding window the table may hold anything: nothing is looked up, nothing reported."""
    cache = _cache([500], 2, 128, 32, 16, dtype, 1)
    q = _queries(new, 8, 128, dtype)
    more = dict(kv_lo=_ints([500 - new + i - 30 for i in range(new)]))
    if new > 1:
        more |= dict(token_offsets=_ints([0, new]), max_tokens=new)
    want, lse = _weighed(cache, q, _ints([500]), **more)
    cache.page_table[:(500 - new - 30) // 16] = -1
    got, _ = _weighed(cache, q, _ints([500]), lse=lse, **more)
    assert _same(got, want) and status.item() == 0 and bool((got > 0).any())


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_wrong_tables_and_lengths(status, dtype):
    from strict_topk_overlap_b200 import paged_eviction
    q = _queries(2, 8, 128, dtype)
    for page, code in ((-1, 2), (10 ** 6, 2)):
        cache = _cache([100, 70], 2, 128, 32, 16, dtype, 2)
        good, lse = _weighed(cache, q, _ints([100, 70]))
        cache.page_table[1] = page
        got, _ = _weighed(cache, q, _ints([100, 70]), lse=lse)
        assert status.item() == code
        assert _same(got[:, 4:], good[:, 4:])  # the other request
        status.zero_()
        cache = _filled([100, 70], 2, 128, 32, 16, dtype, 2)
        cache.page_table[1] = page
        weights = torch.rand((2, 7, 32), device=DEV)
        paged_eviction.evict(cache, weights, _ints([100, 70]), 40)
        assert status.item() == code
        status.zero_()
    cache = _filled([100, 70], 2, 128, 32, 16, dtype, 2)
    got, _ = _weighed(cache, q, _ints([100, 1000]), lse=torch.zeros((2, 8), device=DEV))
    assert status.item() == 5
    status.zero_()
    now, kept = paged_eviction.evict(cache, torch.rand((2, 7, 32), device=DEV), _ints([-5, 1000]), 40)
    assert status.item() == 5 and now.tolist() == [0, 40] and kept[0].eq(-1).all() and int(kept[1].max()) < 96


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_more_tokens_than_promised(status, dtype):
    """A request's tokens past max_tokens are left out and reported; the others' are not."""
    cache = _cache([100, 70], 2, 128, 32, 16, dtype, 3)
    q = _queries(23, 8, 128, dtype)
    more = dict(token_offsets=_ints([0, 20, 23]))
    _, lse = _weighed(cache, q, _ints([100, 70]), **more)
    got, _ = _weighed(cache, q, _ints([100, 70]), lse=lse, max_tokens=4, **more)
    assert status.item() == 3
    lse[4:20] = float("-inf")
    status.zero_()
    want, _ = _weighed(cache, q, _ints([100, 70]), lse=lse, max_tokens=20, **more)
    assert status.item() == 0 and bool(((got - want).abs() <= 1e-5 * want.abs()).all())


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding(dtype):
    """Tokens behind the last request's are nobody's, whatever they and their log-sum-exps hold."""
    cache = _cache([100, 70], 2, 128, 32, 16, dtype, 4)
    q = _queries(30, 8, 128, dtype)
    offsets = _ints([0, 9, 21])
    want, lse = _weighed(cache, q[:21], _ints([100, 70]), token_offsets=offsets, max_tokens=12)
    q[21:] = float("nan")
    got, _ = _weighed(cache, q, _ints([100, 70]), lse=torch.cat((lse, lse.new_full((9, 8), float("nan")))), token_offsets=offsets,
                      max_tokens=12)
    assert _same(got, want)


@gpu
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HALF, 64), (F32, 128)])
@pytest.mark.parametrize("new", [1, 30])
def test_values_that_are_not_finite(dtype, d, new):
    """NaN and infinite keys that some tokens see, and NaN queries: NaN where the definition has it, nowhere else."""
    cache = _cache([200], 2, d, 32, 16, dtype, 5)
    q = _queries(new, 4, d, dtype)
    where = cache.page_table[40 // 16].long()
    cache.k_pages[where, 0, 8] = float("nan")
    cache.k_pages[cache.page_table[90 // 16].long(), 1, 10] = float("inf")
    q[new // 2, 3] = float("nan")
    lse = 5 + torch.rand((new, 4), device=DEV)
    offsets = dict(token_offsets=_ints([0, new]), max_tokens=new) if new > 1 else {}
    got, _ = _weighed(cache, q, _ints([200]), lse=lse, **offsets)
    from oracle import paged_dense as O
    k = O.gather(cache.k_pages, cache.page_table, cache.block_offsets.tolist(), 32, 16, 0, 200)
    pos = list(range(200 - new, 200))
    want, _, _ = E.key_weights(q, k, lse, [0] * new, [p + 1 for p in pos], pos, scale=d ** -0.5)
    got = got.view(2, -1)[:, :200].double()
    assert torch.equal(got.isnan(), want.isnan()) and bool(want.isnan().any())
    live = want.isfinite()
    assert torch.equal(got.isinf(), want.isinf())
    assert bool(((got - want)[live].abs() <= 2.0 ** -14 * want[live]).all())  # (finiteness is what is tested here)


@gpu
def test_the_same_bits_again():
    """Parts of prompts' rows are joined in order, chunks are moved whoever comes first: no bit depends on timing."""
    from strict_topk_overlap_b200 import paged_eviction
    cache = _cache([3000], 2, 128, 32, 16, BF, 6)
    q = _queries(3000, 8, 128, BF)
    more = dict(token_offsets=_ints([0, 3000]), max_tokens=3000)
    first, lse = _weighed(cache, q, _ints([3000]), **more)
    for _ in range(3):
        again, _ = _weighed(cache, q, _ints([3000]), lse=lse, **more)
        assert _same(again, first)
    pools = []
    for _ in range(3):
        cache = _filled([3000], 2, 128, 32, 16, BF, 6)
        paged_eviction.evict(cache, first.clone(), _ints([3000]), 1000, first=4, last=100)
        pools.append((cache.k_pages, cache.v_pages, cache.lo))
    assert all(_same(a, b) for pool in pools[1:] for a, b in zip(pool, pools[0]))


@gpu
def test_captured_and_replayed():
    """One graph of all three, replayed on other lengths, queries and logits, on tensors that stay where they are."""
    from strict_topk_overlap_b200 import paged_attention, paged_eviction, sampling
    from strict_topk_overlap_b200.paged import PagedKVCache
    base = _filled([256, 256], 2, 128, 32, 16, BF, 7)
    weights, out = torch.rand((2, 16, 32), device=DEV), torch.empty((2, 16, 32), device=DEV)
    q, lengths = _queries(2, 8, 128, BF), _ints([200, 100])
    logits, u = torch.randn((2, 999), device=DEV), torch.rand((2,), device=DEV)
    tensors = [base.k_pages, base.v_pages, base.lo, base.hi, weights]

    def step():
        _, lse = paged_attention.attention(q, base, lengths, return_lse=True)
        paged_eviction.accumulate_weights(weights, q, base, lengths, lse)
        now, kept = paged_eviction.evict(base, weights, lengths, 90, first=2, last=3, weights_out=out)
        return now, kept, sampling.sample(logits, u, top_k=20, top_p=0.9)

    saved = [x.clone() for x in tensors]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for lens in ([200, 100], [256, 33], [90, 1]):
        lengths.copy_(_ints(lens))
        q.copy_(_queries(2, 8, 128, BF, seed=sum(lens)))
        logits.copy_(torch.randn((2, 999), generator=torch.Generator(DEV).manual_seed(sum(lens)), device=DEV))
        for x, y in zip(tensors, saved):
            x.copy_(y)
        eager = [x.clone() for x in (*step(), *tensors, out)]
        for x, y in zip(tensors, saved):
            x.copy_(y)
        out.zero_()
        graph.replay()
        assert all(_same(a, b) for a, b in zip((*results, *tensors, out), eager)), lens
    assert isinstance(base, PagedKVCache)


@gpu
def test_two_streams():
    """Two evictions and two weighings at once, each on its own stream and cache, and sampling beside them."""
    from strict_topk_overlap_b200 import paged_eviction, sampling
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    x, u = torch.randn((4, 30000), device=DEV), torch.rand((4,), device=DEV)
    q = _queries(64, 8, 128, BF)
    more = dict(token_offsets=_ints([0, 64]), max_tokens=64)

    def work(cache, w):
        _weighed(cache, q, _ints([5000]), weights=w, lse=torch.full((64, 8), 8.0, device=DEV), **more)
        now, kept = paged_eviction.evict(cache, w, _ints([5000]), 2000, last=10)
        return [cache.k_pages, cache.v_pages, cache.lo, w, kept, sampling.sample(x, u, top_p=0.8)]

    def fresh(i):
        return _filled([5000], 2, 128, 32, 16, BF, 8 + i), torch.rand((2, 157, 32), generator=torch.Generator(DEV).manual_seed(i), device=DEV)

    want = [work(*fresh(i)) for i in range(2)]
    inputs = [fresh(i) for i in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            got.append(work(*inputs[i]))
    torch.cuda.synchronize()
    assert all(_same(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@gpu
@pytest.mark.parametrize("dtype,shift", [(BF, 1), (HALF, 2), (F32, 1), (BF, 8)])
def test_pools_off_a_boundary(dtype, shift):
    """Pools that begin at any element: other kernels and other pieces, the same values."""
    from strict_topk_overlap_b200 import paged_eviction
    cache = _filled([300], 2, 64, 32, 16, dtype, 9)
    moved = _filled([300], 2, 64, 32, 16, dtype, 9)
    for name in ("k_pages", "v_pages"):
        x = getattr(cache, name)
        room = torch.empty((x.numel() + shift,), dtype=dtype, device=DEV)
        room[shift:].copy_(x.flatten())
        setattr(moved, name, room[shift:].view(x.shape))
    q = _queries(1, 4, 64, dtype)
    a, lse = _weighed(cache, q, _ints([300]))
    b, _ = _weighed(moved, q, _ints([300]), lse=lse)
    assert bool(((a - b).abs() <= 1e-5 * a).all())
    for c in (cache, moved):
        paged_eviction.evict(c, a.clone(), _ints([300]), 77, first=1, last=5)
    assert _same(cache.k_pages, moved.k_pages) and _same(cache.v_pages, moved.v_pages) and _same(cache.lo, moved.lo)


@gpu
def test_shared_prefix_stays():
    """Requests behind one prefix, its pages in all their tables: protected by `first`, they are not written."""
    from strict_topk_overlap_b200 import paged_eviction
    cache = _cache([400, 300, 350], 2, 128, 32, 16, BF, 10, shared=128)
    pages = cache.page_table[:8].long()
    before = cache.k_pages[pages].clone(), cache.v_pages[pages].clone()
    w = torch.rand((2, cache.page_table.numel() // 2, 32), device=DEV)
    now, kept = paged_eviction.evict(cache, w, _ints([400, 300, 350]), 200, first=128, last=8)
    assert now.tolist() == [200] * 3 and torch.equal(kept[..., :128], torch.arange(128, dtype=torch.int32, device=DEV).expand(3, 2, 128))
    assert _same(cache.k_pages[pages], before[0]) and _same(cache.v_pages[pages], before[1])


@gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements: tokens in its last pages are read and moved like any other."""
    from strict_topk_overlap_b200 import paged, paged_eviction
    pages, hkv, page, d = 140000, 8, 16, 128
    k = torch.zeros((pages, hkv, page, d), dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator(DEV).manual_seed(11)
    table = torch.arange(pages - 64, pages, dtype=torch.int32, device=DEV)
    k[-64:], v[-64:] = (torch.randn((64, hkv, page, d), generator=g, device=DEV).to(BF) for _ in range(2))
    none = torch.empty((hkv, 0, d), device=DEV)
    far = paged.PagedKVCache(k, v, table, _ints([0, 32]), none, none, 32, 16, 32)
    near = paged.PagedKVCache(k[-64:].clone(), v[-64:].clone(), table - (pages - 64), _ints([0, 32]), none, none, 32, 16, 32)
    q = _queries(1, 8, d, BF)
    a, lse = _weighed(near, q, _ints([1000]))
    b, _ = _weighed(far, q, _ints([1000]), lse=lse)
    assert _same(a, b)
    for c in (near, far):
        paged_eviction.evict(c, a.clone(), _ints([1000]), 300)
    assert _same(far.k_pages[-64:].contiguous(), near.k_pages) and _same(far.v_pages[-64:].contiguous(), near.v_pages)
