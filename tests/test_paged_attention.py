"""Dense paged attention against its definition in 64 bits.

With u the output type's rounding (2^-8, 2^-11, 2^-24 relative), A the largest
magnitude that a score of noticeable weight is summed from (scale |q|.|k| plus
the bias) and V the head's largest |v|, an output is off by at most
  u |o|                      its own rounding,
  u V                        16-bit types: weights rounded to the type for the
                             tensor cores (none in FP32),
  2 ds V                     scores off by ds: weights change by a factor
                             e^ds, numerator and denominator,
  c 2^-24 V                  sums of the weights (pairwise over at most 2^14
                             keys here, c = 64 leaves room for the splits),
with ds = (D + 16) 2^-24 A for a dot product of D terms, its scaling, cap and
bias, plus 1e-4 for the 16-bit forms, whose exponentials and caps may be
polynomials of that accuracy (under half of f16's rounding of a weight). The
log-sum-exp is off by at most ds + 64 * 2^-24 + 2^-22 |lse|."""
from __future__ import annotations

import pytest
import torch

from oracle import paged_dense as O

gpu = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _cache(lengths, hkv, d, block, page, dtype, seed, *, shared=0, room=0):
    """A filled pool; slots past a request's tokens hold NaN, as memory never written may."""
    from strict_topk_overlap_b200 import paged
    g = torch.Generator(DEV).manual_seed(seed)
    ppb = block // page
    blocks = [max(1, -(-(n + room) // block)) for n in lengths]
    pre = shared // block
    own = [n - pre for n in blocks]
    pages = (pre + sum(own)) * ppb
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    rows, at = [], pre
    for n in own:
        rows += [order[:pre * ppb], order[at * ppb:(at + n) * ppb]]
        at += n
    table = torch.cat(rows)
    k = torch.randn((pages, hkv, page, d), generator=g, device=DEV)
    k = (k + 0.5 * torch.randn((pages, hkv, 1, d), generator=g, device=DEV)).to(dtype)
    v = torch.randn((pages, hkv, page, d), generator=g, device=DEV).to(dtype)
    offsets = [0]
    for n in blocks:
        offsets.append(offsets[-1] + n)
    for r, n in enumerate(lengths):
        j = torch.arange(n, blocks[r] * block, device=DEV)
        pg = table[offsets[r] * ppb + j // page].long()
        k[pg, :, j % page] = float("nan")
        v[pg, :, j % page] = float("nan")
    none = torch.empty((hkv, 0, d), device=DEV)
    return paged.PagedKVCache(k, v, table, torch.tensor(offsets, dtype=torch.int32, device=DEV), none, none, block,
                              page, max(blocks))


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _compare(q, cache, lengths, new, lo, hi, got, lse, softcap, slopes, scale, seen=None):
    dtype, d = q.dtype, q.shape[2]
    off = cache.block_offsets.tolist()
    start = 0
    for r, (n, length) in enumerate(zip(new, lengths)):
        if n == 0:
            continue
        rows = slice(start, start + n)
        k = O.gather(cache.k_pages, cache.page_table, off, cache.block_size, cache.page_size, r, length)
        v = O.gather(cache.v_pages, cache.page_table, off, cache.block_size, cache.page_size, r, length)
        pos = list(range(length - n, length))
        a = lo[rows] if lo is not None else [0] * n
        b = hi[rows] if hi is not None else [p + 1 for p in pos]
        want, wlse, size, vmax = O.attention(q[rows], k, v, a, b, pos, scale=scale, softcap=softcap, slopes=slopes)
        ds = (d + 16) * 2.0 ** -24 * size + (1e-4 if dtype != torch.float32 else 0.0)
        u = UNIT[dtype]
        tol = u * want.abs() + ((0.0 if dtype == torch.float32 else u) + 2 * ds + 64 * 2.0 ** -24)[..., None] * vmax[..., None]
        bad = (got[rows].double() - want).abs() > tol
        bad |= got[rows].isnan() != want.isnan()
        assert not bool(bad.any()), (r, bad.nonzero()[:5].tolist(), got[rows][bad][:5], want[bad][:5])
        if lse is not None:
            live = wlse != float("-inf")
            assert torch.equal(lse[rows] == float("-inf"), ~live)
            off_by = (lse[rows].double() - wlse)[live].abs()
            assert bool((off_by <= (ds + 64 * 2.0 ** -24 + 2.0 ** -22 * wlse.abs())[live]).all()), off_by.max()
        start += n


def _run(lengths, new, hq, hkv, d, block, page, dtype, seed, *, mask="causal", softcap=0.0, biased=False, scale=None,
         strided=False, prefix=0, **more):
    from strict_topk_overlap_b200 import paged_attention
    cache = _cache(lengths, hkv, d, block, page, dtype, seed, shared=prefix)
    g = torch.Generator(DEV).manual_seed(seed + 1)
    t = sum(new)
    q = torch.randn((t, hq + (3 if strided else 0), d), generator=g, device=DEV).to(dtype)
    if strided:
        q = q[:, 1:hq + 1]
    lo = hi = None
    pos = [p for n, length in zip(new, lengths) for p in range(length - n, length)]
    if mask == "window":
        lo = [max(0, p - 36) for p in pos]
    elif mask == "documents":
        lo = [p // 29 * 29 for p in pos]
    elif mask == "prefix":
        hi = [max(p + 1, 75) for p in pos]
    elif mask == "odd":  # empty intervals, ends beyond the cache, negative starts, single keys
        lo = [(-4, 7, p, 30, p + 1)[i % 5] for i, p in enumerate(pos)]
        hi = [(1 << 30, 7, p + 1, 20, p + 1)[i % 5] for i, p in enumerate(pos)]
    offsets = None
    if any(n != 1 for n in new):
        offsets = _ints([0] + list(torch.tensor(new).cumsum(0)))
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if biased else None
    args = dict(token_offsets=offsets, max_tokens=max(new), kv_lo=None if lo is None else _ints(lo),
                kv_hi=None if hi is None else _ints(hi), softcap=softcap, slopes=slopes, scale=scale, return_lse=True)
    args.update(more)
    if prefix:
        out, lse = paged_attention.shared_prefix_attention(q, cache, _ints(lengths), prefix, **args)
    else:
        out, lse = paged_attention.attention(q, cache, _ints(lengths), **args)
    _compare(q, cache, lengths, new, lo, hi, out, lse, softcap, slopes, scale or d ** -0.5)
    return out


SHAPES = [  # hq, hkv, d, block, page
    (8, 2, 128, 32, 16), (4, 4, 64, 64, 32), (24, 2, 128, 32, 32), (5, 1, 64, 32, 16), (16, 1, 128, 128, 128),
    (40, 2, 64, 16, 16), (6, 2, 96, 24, 8), (3, 1, 40, 6, 3), (4, 2, 256, 32, 16), (2, 1, 320, 16, 16)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_single_tokens(dtype, shape):
    """One token for each of several requests of 1 to 700 tokens, some ending inside a page."""
    _run([1, 700, 33, 64, 257, 16], [1] * 6, *shape, dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_prompts(dtype, shape):
    """Ragged prompts and pieces of prompts, one request without new tokens."""
    _run([130, 1, 90, 20, 200], [130, 1, 37, 0, 5], *shape, dtype, 2)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", ["window", "documents", "prefix", "odd"])
@pytest.mark.parametrize("new", [[1, 1, 1], [150, 40, 3]])
def test_masks(dtype, mask, new):
    for shape in ((8, 2, 128, 32, 16), (6, 2, 96, 24, 8), (12, 1, 64, 32, 32)):
        _run([150, 290, 80], new, *shape, dtype, 3, mask=mask)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1], [140, 33]])
@pytest.mark.parametrize("softcap,biased,scale", [(50.0, False, None), (0.0, True, None), (2.0, True, 0.7),
                                                  (0.25, False, 3.0)])
def test_scores(dtype, new, softcap, biased, scale):
    for shape in ((8, 2, 128, 32, 16), (4, 2, 64, 32, 16), (6, 2, 96, 24, 8)):
        _run([300, 65], new, *shape, dtype, 4, softcap=softcap, biased=biased, scale=scale, mask="prefix")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_long_and_split(dtype):
    """Key ranges that are cut into many parts and joined, and many requests of very different lengths."""
    _run([9000], [1], 8, 2, 128, 32, 16, dtype, 5)
    _run([9001, 1, 17, 5000, 300], [1] * 5, 4, 1, 64, 32, 16, dtype, 6)
    _run([5003], [9], 8, 2, 128, 32, 16, dtype, 7, biased=True)
    _run(list(range(1, 140)), [1] * 139, 2, 1, 64, 32, 16, dtype, 8)
    _run([700], [300], 4, 1, 128, 32, 16, dtype, 9, strided=True)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1] * 4, [3, 3, 3, 3], [40, 1, 0, 7]])
def test_shared_prefix(dtype, new):
    for shape in ((8, 2, 128, 32, 16), (4, 4, 64, 32, 32), (24, 2, 128, 32, 16), (6, 2, 96, 24, 8)):
        block = shape[3]
        prefix = 7 * block
        lengths = [prefix + max(n, e) for n, e in zip(new, (1, 100, 33, 7))]
        _run(lengths, new, *shape, dtype, 10, prefix=prefix)
        _run(lengths, new, *shape, dtype, 11, prefix=prefix, mask="window", softcap=5.0)
        _run(lengths, new, *shape, dtype, 12, prefix=prefix, mask="prefix", biased=True)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_shared_prefix_many_rows(dtype):
    """Enough rows behind the prefix for full tensor-core tiles."""
    _run([640 + i for i in range(1, 41)], [1] * 40, 32, 2, 128, 32, 16, dtype, 13, prefix=640)
    _run([1280 + i % 3 + 4 for i in range(12)], [4] * 12, 8, 1, 64, 32, 16, dtype, 14, prefix=1280)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1], [90, 64]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_places_do_not_matter(dtype, new, bad):
    """A key that a token does not see may hold anything: a packed document next to one that overflowed."""
    from strict_topk_overlap_b200 import paged_attention
    for hq, hkv, d, block, page in ((8, 2, 128, 32, 16), (6, 2, 96, 24, 8), (4, 4, 64, 32, 16)):
        lengths = [150, 100]
        cache = _cache(lengths, hkv, d, block, page, dtype, 20)
        q = torch.randn((sum(new), hq, d), generator=torch.Generator(DEV).manual_seed(21), device=DEV).to(dtype)
        pos = [p for n, length in zip(new, lengths) for p in range(length - n, length)]
        lo = [p // 75 * 75 for p in pos]
        args = dict(token_offsets=None if max(new) == 1 else _ints([0, new[0], sum(new)]), max_tokens=max(new),
                    kv_lo=_ints(lo))
        clean = paged_attention.attention(q, cache, _ints(lengths), **args)
        off, ppb = cache.block_offsets.tolist(), block // page
        for j in (3, 40, 74):  # in the first document of request 0
            pg = int(cache.page_table[off[0] * ppb + j // page])
            cache.k_pages[pg, :, j % page] = bad
            cache.v_pages[pg, :, j % page] = bad
        out = paged_attention.attention(q, cache, _ints(lengths), **args)
        unseen = torch.tensor([r > 0 or a >= 75 for r, n in enumerate(new) for a in lo[sum(new[:r]):sum(new[:r]) + n]],
                              device=DEV)
        assert bool(unseen.any())
        _compare_equal(out[unseen], clean[unseen], dtype)
        # Rows that see a NaN or infinite key are not finite numbers made up by the mask.
        for i, p in enumerate(pos[:new[0]]):
            if lo[i] == 0 and p >= 3 and bad != bad:
                assert bool(out[i].isnan().all())


def _compare_equal(a, b, dtype):
    """Rows of the same inputs: equal up to the order of their sums."""
    assert bool(a.isfinite().all())
    tol = 4 * UNIT[dtype] * 6
    assert float((a.double() - b.double()).abs().max()) <= tol


@gpu
def test_scores_of_the_types_lowest_value():
    """Keys whose scores are far below the others', or all equal and huge, keep a finite softmax."""
    from strict_topk_overlap_b200 import paged_attention
    for dtype, big in ((torch.float32, 1e18), (torch.bfloat16, 1e18), (torch.float16, 200.0)):
        for new in (1, 130):
            cache = _cache([200], 2, 64, 32, 16, dtype, 30)
            cache.k_pages.fill_(-big)
            q = torch.full((new, 4, 64), big, dtype=dtype, device=DEV)
            out, lse = paged_attention.attention(q, cache, _ints([200]), max_tokens=new, return_lse=True,
                                                 token_offsets=None if new == 1 else _ints([0, new]))
            v = O.gather(cache.v_pages, cache.page_table, cache.block_offsets.tolist(), 32, 16, 0, 200)
            want = v[:, :200].double().mean(1)  # all scores equal: the mean
            got = out[-1].view(2, 2, 64).double()
            assert float((got - want[:, None]).abs().max()) <= 4 * UNIT[dtype] * 5
            assert bool(lse.isfinite().all())


def _scores_along(pattern, n):
    """Scores of n keys, in nats, that move far from one run of keys to the next."""
    j = torch.arange(n, device=DEV, dtype=torch.float32)
    if pattern == "ramp":
        return 0.7 * (j - n / 2)
    if pattern == "fall":
        return -0.7 * j
    if pattern == "jump":  # one key far above all before it, more than the types' range of weights
        return torch.where(j == 300, 150.0, torch.where(j > 300, 20.0, 0.0))
    if pattern == "halves":  # every second run of 64 keys far above the other
        return torch.where(j % 128 >= 64, 110.0, 0.0) + 0.01 * j
    return torch.where(j < n - 3, -400.0, 300.0)  # "last": all weight on the last keys


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pattern", ["ramp", "fall", "jump", "halves", "last"])
@pytest.mark.parametrize("new", [1, 40, 200])
def test_scores_that_move(dtype, pattern, new):
    """The running maximum, wherever a kernel keeps it, follows scores that grow by hundreds between runs of keys."""
    from strict_topk_overlap_b200 import paged_attention
    for hq, hkv, d, block, page in ((8, 2, 128, 32, 16), (4, 2, 64, 32, 32), (2, 1, 96, 32, 16)):
        n = 700
        cache = _cache([n], hkv, d, block, page, dtype, 70)
        along = _scores_along(pattern, n) * d ** 0.5 / 16
        j = torch.arange(n, device=DEV)
        pg = cache.page_table[j // page].long()
        cache.k_pages[pg, :, j % page] *= 0.25
        cache.k_pages[pg, :, j % page, 0] = along.to(dtype)[:, None].expand(-1, hkv)
        q = (0.25 * torch.randn((new, hq, d), generator=torch.Generator(DEV).manual_seed(71), device=DEV)).to(dtype)
        q[..., 0] = 16.0
        offsets = None if new == 1 else _ints([0, new])
        for softcap, slopes in ((0.0, None), (300.0, None), (0.0, torch.full((hq,), 4.0, device=DEV))):
            out, lse = paged_attention.attention(q, cache, _ints([n]), token_offsets=offsets, max_tokens=new,
                                                 softcap=softcap, slopes=slopes, return_lse=True)
            _compare(q, cache, [n], [new], None, None, out, lse, softcap, slopes, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_steep_biases(dtype):
    """Biases that grow by hundreds from tile to tile, ranges that end inside a tile, tokens far behind the keys they see."""
    from strict_topk_overlap_b200 import paged_attention
    for hq, hkv, d, block, page in ((8, 2, 128, 32, 16), (4, 2, 64, 32, 32)):
        for n, new, seen in ((1000, 70, 1000), (1000, 70, 545), (1000, 40, 640 + 1), (1500, 300, 900)):
            cache = _cache([n], hkv, d, block, page, dtype, 90)
            q = torch.randn((new, hq, d), generator=torch.Generator(DEV).manual_seed(91), device=DEV).to(dtype)
            pos = list(range(n - new, n))
            hi = [min(p + 1, seen) for p in pos]
            slopes = torch.tensor([(0.84, 3.0, 0.1, 0.5)[h % 4] for h in range(hq)], device=DEV)
            out, lse = paged_attention.attention(q, cache, _ints([n]), token_offsets=_ints([0, new]), max_tokens=new,
                                                 kv_hi=_ints(hi), slopes=slopes, return_lse=True)
            _compare(q, cache, [n], [new], None, hi, out, lse, 0.0, slopes, d ** -0.5)


@gpu
def test_offsets_past_32_bits():
    """Pages whose elements lie beyond 2^31 of their pool: the append writes them, every attention form reads them."""
    from strict_topk_overlap_b200 import paged, paged_append, paged_attention
    pages, hkv, page, d = 140000, 8, 16, 128  # 2.3e9 elements
    pool = [torch.empty((pages, hkv, page, d), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    table = (pages - 1 - torch.arange(20, device=DEV)).to(torch.int32)
    none = torch.empty((hkv, 0, d), device=DEV)
    cache = paged.PagedKVCache(pool[0], pool[1], table, _ints([0, 10]), none, none, 32, page, 10)
    g = torch.Generator(DEV).manual_seed(80)
    k, v = (torch.randn((300, hkv, d), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    paged_append.append_tokens(cache, k, v, _ints([0]), token_offsets=_ints([0, 300]))
    got = pool[0][table.long()].transpose(0, 1).reshape(hkv, -1, d)[:, :300].transpose(0, 1)
    assert torch.equal(got, k)
    q = torch.randn((300, 16, d), generator=g, device=DEV).to(torch.bfloat16)
    for new in (1, 300):
        x = q[300 - new:]
        more = dict(token_offsets=None if new == 1 else _ints([0, new]), max_tokens=new, return_lse=True)
        out, lse = paged_attention.attention(x, cache, _ints([300]), **more)
        _compare(x, cache, [300], [new], None, None, out, lse, 0.0, None, d ** -0.5)
    out, lse = paged_attention.shared_prefix_attention(q[:1], cache, _ints([300]), 160, return_lse=True)
    _compare(q[:1], cache, [300], [1], None, None, out, lse, 0.0, None, d ** -0.5)


@gpu
def test_streams_graphs_and_workspaces():
    from strict_topk_overlap_b200 import paged_attention
    lengths = [500, 77, 1200]
    cache = _cache(lengths, 2, 128, 32, 16, torch.bfloat16, 40)
    q = torch.randn((3, 8, 128), device=DEV).to(torch.bfloat16)
    at = _ints(lengths)
    want = paged_attention.attention(q, cache, at)
    ws = paged_attention.attention_workspace(cache, 3, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = paged_attention.attention(q, cache, at, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = paged_attention.attention(q, cache, at, workspace=ws)
    shorter = _ints([300, 2, 900])
    at.copy_(shorter)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, paged_attention.attention(q, cache, shorter))
    assert torch.equal(held, paged_attention.attention(q, cache, shorter))  # the same bits every time
    with pytest.raises(RuntimeError, match="workspace"):
        paged_attention.attention(q, cache, at, workspace=ws[:16])
    with pytest.raises(RuntimeError, match="16-byte"):
        paged_attention.attention(q, cache, at, workspace=torch.cat((ws, ws))[8:])


@gpu
@pytest.mark.parametrize("new", [1, 130])
def test_unaligned_tensors(new):
    """Queries, pools and outputs that start off a 16-byte boundary take another kernel, not another result."""
    import ctypes

    from strict_topk_overlap_b200 import _lib as L
    from strict_topk_overlap_b200 import paged, paged_attention
    cache = _cache([200], 2, 64, 32, 16, torch.bfloat16, 52)

    def shifted(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape)
        return y.copy_(x)

    q = torch.randn((new, 4, 64), device=DEV).to(torch.bfloat16)
    off = paged.PagedKVCache(shifted(cache.k_pages), shifted(cache.v_pages), cache.page_table, cache.block_offsets,
                             cache.lo, cache.hi, 32, 16, cache.max_blocks)
    more = dict(max_tokens=new, token_offsets=None if new == 1 else _ints([0, new]), return_lse=True)
    for x, c in ((shifted(q), cache), (q, off)):
        out, lse = paged_attention.attention(x, c, _ints([200]), **more)
        _compare(q, cache, [200], [new], None, None, out, lse, 0.0, None, 64 ** -0.5)
    # An output off its boundary, through the C entry point.
    out = shifted(torch.zeros_like(q))
    longest = cache.max_blocks * 32
    kv, offsets = cache.packed_kv(2, 64), None if new == 1 else _ints([0, new])
    need = L.load().stk_paged_attention_workspace_bytes(kv, 1, new, 4, int(new > 1), new, longest, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    length = _ints([200])
    rc = L.load().stk_paged_attention(kv, cache.k_pages.shape[0], q.data_ptr(), q.stride(0), q.stride(1), 1, new, 4,
                                      length.data_ptr(), L.ptr(offsets), new, longest, 0, None, out.data_ptr(), None,
                                      ws.data_ptr(), need, None, ctypes.c_void_p(L.stream_of(q)))
    assert rc == 0
    _compare(q, cache, [200], [new], None, None, out, None, 0.0, None, 64 ** -0.5)


@gpu
def test_bad_data_is_reported():
    from strict_topk_overlap_b200 import _lib, paged_attention
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for new in (1, 130):
        cache = _cache([200], 2, 64, 32, 16, torch.bfloat16, 50)
        q = torch.randn((new, 4, 64), device=DEV).to(torch.bfloat16)
        more = dict(max_tokens=new, token_offsets=None if new == 1 else _ints([0, new]))
        try:
            _lib.set_status_tensor(status)
            status.zero_()
            paged_attention.attention(q, cache, _ints([10 ** 6]), **more)
            assert int(status) == 5
            status.zero_()
            cache.page_table[3] = -7
            paged_attention.attention(q, cache, _ints([200]), **more)
            assert int(status) == 2
        finally:
            _lib.set_status_tensor(None)


@gpu
@pytest.mark.parametrize("offsets,new", [([0, 9, 4], 1), ([0, 2, 900], 1), ([-5, 2, 6], 1), ([0, 400, 500], 130),
                                         ([0, 4, 6], 1)])
def test_bad_offsets_and_bounds_are_reported(offsets, new):
    """Offsets that leave the packed tokens, and more tokens than max_tokens: cut, reported, nothing else touched."""
    from strict_topk_overlap_b200 import _lib, paged_append, paged_attention
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = _cache([200, 300], 2, 64, 32, 16, torch.bfloat16, 51)
    t = 6 if new == 1 else 260
    q = torch.randn((t, 8, 64), device=DEV).to(torch.bfloat16)
    try:
        _lib.set_status_tensor(status)
        paged_attention.attention(q, cache, _ints([200, 300]), token_offsets=_ints(offsets), max_tokens=new)
        assert int(status) == 3
        if offsets != [0, 4, 6]:
            status.zero_()
            kv = q[:, :2].contiguous()
            paged_append.append_tokens(cache, kv, kv, _ints([10, 20]), token_offsets=_ints(offsets))
            assert int(status) == 3
    finally:
        _lib.set_status_tensor(None)
    torch.cuda.synchronize()


@gpu
def test_refusals():
    from strict_topk_overlap_b200 import paged_attention
    cache = _cache([64, 64], 2, 64, 32, 16, torch.bfloat16, 60)
    q = torch.randn((2, 4, 64), device=DEV).to(torch.bfloat16)
    at = _ints([64, 64])
    call = paged_attention.attention
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(lengths=at[:1]),
                dict(lengths=at.long()), dict(q=q[:1]), dict(kv_lo=at[:1]), dict(kv_hi=at.long()), dict(softcap=-1.0),
                dict(scale=0.0), dict(slopes=torch.ones(3, device=DEV)), dict(slopes=torch.ones(4)),
                dict(token_offsets=at)):
        args = dict(q=q, lengths=at)
        args.update(bad)
        with pytest.raises(ValueError):
            call(args.pop("q"), cache, args.pop("lengths"), **args)
    for prefix in (-16, 8, 96):
        with pytest.raises(ValueError):
            paged_attention.shared_prefix_attention(q, cache, at, prefix)
    empty = paged_attention.attention(q[:0], cache, at, token_offsets=_ints([0, 0, 0]))
    assert empty.shape == (0, 4, 64)
