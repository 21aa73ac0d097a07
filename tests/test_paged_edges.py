"""Dense paged attention where values, lengths and tables are at their edges:
huge values and NaN at seen and unseen keys, unfilled pages, tokens of no
request. Outputs that an edge must not touch are compared bit for bit with
those of the same call without it; others with the 64-bit definition and the
tolerances of test_paged_attention.py."""
from __future__ import annotations

import pytest
import torch

from oracle import paged_dense as O
from test_paged_attention import DEV, TYPES, UNIT, _cache, _compare, _compare_equal, _ints

gpu = pytest.mark.gpu
TILED = [(8, 2, 128, 32, 16), (4, 4, 64, 32, 16)]  # hq, hkv, d, block, page that the tensor-core kernels take


def _queries(new, hq, d, dtype, seed):
    return torch.randn((new, hq, d), generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


def _at(cache, r, j):
    """Pages and slots of key tokens j (an int tensor) of request r."""
    ppb = cache.block_size // cache.page_size
    first = int(cache.block_offsets[r]) * ppb
    return cache.page_table[first + j // cache.page_size].long(), j % cache.page_size


def _span(a, b):
    return torch.arange(a, b, device=DEV)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", TILED)
@pytest.mark.parametrize("new", [1, 4, 200])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_unseen_values_near_the_types_limit(dtype, shape, new, sign):
    """A key outside a row's interval weighs exactly nothing: its value may be as large as the type holds."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    cache = _cache([300], hkv, d, block, page, dtype, 100)
    q = _queries(new, hq, d, dtype, 101)
    pos = list(range(300 - new, 300))
    split = [(p - 80) // 7 * 7 for p in pos]  # a first document of 14 to 217 keys
    for scores in (dict(), dict(softcap=20.0), dict(slopes=torch.full((hq,), 0.05, device=DEV))):
        args = dict(token_offsets=None if new == 1 else _ints([0, new]), max_tokens=new, return_lse=True, **scores)
        for lo, hi, keys in ((split, None, _span(0, min(split))), (None, [240] * new, _span(240, 300)),
                             (None, None, _span(300 - new + 1, 300))):
            if keys.numel() == 0:
                continue
            more = dict(args, kv_lo=None if lo is None else _ints(lo), kv_hi=None if hi is None else _ints(hi))
            clean, clean_lse = paged_attention.attention(q, cache, _ints([300]), **more)
            at = _at(cache, 0, keys)
            held = cache.v_pages[at[0], :, at[1]].clone()
            cache.v_pages[at[0], :, at[1]] = sign * {torch.float16: 65504.0}.get(dtype, 3e38)
            out, lse = paged_attention.attention(q, cache, _ints([300]), **more)
            cache.v_pages[at[0], :, at[1]] = held
            first = int(keys[0])
            blind = torch.tensor([(hi is not None) or (lo is not None) or p < first for p in pos], device=DEV)
            assert bool(blind.any())
            assert torch.equal(out[blind], clean[blind])
            assert torch.equal(lse, clean_lse)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", TILED)
@pytest.mark.parametrize("new", [1, 200])
@pytest.mark.parametrize("biased", [False, True])
def test_seen_nan_keys_are_not_lost(dtype, shape, new, biased):
    """A NaN in one key (its value is a number) makes every row that sees it NaN, wherever in a run of keys it lies,
    and no other row."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    cache = _cache([300], hkv, d, block, page, dtype, 102)
    q = _queries(new, hq, d, dtype, 103)
    args = dict(token_offsets=None if new == 1 else _ints([0, new]), max_tokens=new, return_lse=True,
                slopes=torch.full((hq,), 0.05, device=DEV) if biased else None)
    clean, _ = paged_attention.attention(q, cache, _ints([300]), **args)
    pos = _span(300 - new, 300)
    for j in list(range(32, 48)) + [150, 215, 290, 299]:
        pg, slot = _at(cache, 0, _span(j, j + 1))
        held = cache.k_pages[pg, :, slot, 5].clone()
        cache.k_pages[pg, :, slot, 5] = float("nan")
        out, lse = paged_attention.attention(q, cache, _ints([300]), **args)
        cache.k_pages[pg, :, slot, 5] = held
        sees = pos >= j
        assert bool(out[sees].isnan().all()) and bool(lse[sees].isnan().all()), j
        if bool((~sees).any()):
            _compare_equal(out[~sees], clean[~sees], dtype)


FORMS = TILED + [(6, 2, 96, 24, 8)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FORMS)
@pytest.mark.parametrize("new,prefix", [(1, 0), (4, 0), (200, 0), (1, 240), (40, 240)])
def test_nan_query(dtype, shape, new, prefix):
    """A query row that is NaN comes out as NaN, not as one that sees no keys; the others do not change."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    prefix = prefix // block * block
    cache = _cache([300, 400], hkv, d, block, page, dtype, 104, shared=prefix)
    q = _queries(2 * new, hq, d, dtype, 105)
    args = dict(token_offsets=None if new == 1 else _ints([0, new, 2 * new]), max_tokens=new, return_lse=True)

    def call(q):
        if prefix:
            return paged_attention.shared_prefix_attention(q, cache, _ints([300, 400]), prefix, **args)
        return paged_attention.attention(q, cache, _ints([300, 400]), **args)

    clean, clean_lse = call(q)
    broken = torch.zeros((2 * new, hq), dtype=torch.bool, device=DEV)
    broken[0, 0] = broken[-1, hq - 1] = broken[new // 2, hq // 2] = True
    q[broken] = float("nan")
    out, lse = call(q)
    assert bool(out[broken].isnan().all()) and bool(lse[broken].isnan().all())
    _compare_equal(out[~broken], clean[~broken], dtype)
    assert float((lse - clean_lse)[~broken].abs().max()) <= 1e-3


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FORMS)
@pytest.mark.parametrize("new", [1, 4, 200])
def test_only_nan_keys(dtype, shape, new):
    """Rows whose only visible keys score NaN are NaN; rows that see no key at all are zero."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    cache = _cache([300], hkv, d, block, page, dtype, 106)
    q = _queries(new, hq, d, dtype, 107)
    pos = list(range(300 - new, 300))
    for width in (0, 1, 30):
        keys = _span(299 - new - 30, 300)
        at = _at(cache, 0, keys)
        held = cache.k_pages[at[0], :, at[1]].clone()
        cache.k_pages[at[0], :, at[1], 3] = float("nan")
        out, lse = paged_attention.attention(q, cache, _ints([300]), max_tokens=new, return_lse=True,
                                             token_offsets=None if new == 1 else _ints([0, new]),
                                             kv_lo=_ints([p + 1 - width for p in pos]))
        cache.k_pages[at[0], :, at[1]] = held
        if width:
            assert bool(out.isnan().all()) and bool(lse.isnan().all())
        else:
            assert not bool(out.any()) and bool((lse == float("-inf")).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FORMS)
@pytest.mark.parametrize("new", [1, 130])
def test_a_part_of_nan_keys_does_not_vanish(dtype, shape, new):
    """Long ranges are cut into parts and tiles into halves: one whose keys are all NaN still makes the row NaN."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    cache = _cache([6000], hkv, d, block, page, dtype, 108)
    q = _queries(new, hq, d, dtype, 109)
    for a, b in ((0, 64), (64, 128), (3000, 3700), (5760, 5824)):
        at = _at(cache, 0, _span(a, b))
        held = cache.k_pages[at[0], :, at[1]].clone()
        cache.k_pages[at[0], :, at[1], 1] = float("nan")
        out, lse = paged_attention.attention(q, cache, _ints([6000]), max_tokens=new, return_lse=True,
                                             token_offsets=None if new == 1 else _ints([0, new]))
        cache.k_pages[at[0], :, at[1]] = held
        assert bool(out.isnan().all()) and bool(lse.isnan().all())


ROOMY = TILED + [(8, 2, 128, 128, 16), (4, 1, 64, 256, 32), (24, 2, 128, 256, 256)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ROOMY)
@pytest.mark.parametrize("new", [[1] * 4, [130, 90, 1, 44]])
def test_unfilled_pages_change_nothing(dtype, shape, new):
    """NaN in every slot past the tokens, whole pages of it, gives the bits that zeros there give: no row leaves its
    fast path for what it does not see."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    lengths = [130, 200, 1, 300]
    cache = _cache(lengths, hkv, d, block, page, dtype, 110)
    q = _queries(sum(new), hq, d, dtype, 111)
    at = torch.tensor([0] + new).cumsum(0).tolist()
    args = dict(token_offsets=None if max(new) == 1 else _ints(at), max_tokens=max(new), return_lse=True)
    for scores in (dict(), dict(softcap=20.0, slopes=torch.full((hq,), 0.1, device=DEV))):
        got = paged_attention.attention(q, cache, _ints(lengths), **args, **scores)
        held = cache.k_pages, cache.v_pages
        cache.k_pages, cache.v_pages = held[0].nan_to_num(0.0), held[1].nan_to_num(0.0)
        want = paged_attention.attention(q, cache, _ints(lengths), **args, **scores)
        cache.k_pages, cache.v_pages = held
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ROOMY[:3])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_unfilled_pages_behind_a_prefix(dtype, shape, new):
    """The pages behind a shared prefix that ends inside a tile of keys belong to request 0 alone, filled or not."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    prefix = 9 * block
    lengths = [prefix + new, prefix + new + 3]
    cache = _cache(lengths, hkv, d, block, page, dtype, 112, shared=prefix, room=2 * block)
    q = _queries(2 * new, hq, d, dtype, 113)
    args = dict(token_offsets=None if new == 1 else _ints([0, new, 2 * new]), max_tokens=new, return_lse=True)
    got = paged_attention.shared_prefix_attention(q, cache, _ints(lengths), prefix, **args)
    cache.k_pages, cache.v_pages = cache.k_pages.nan_to_num(0.0), cache.v_pages.nan_to_num(0.0)
    want = paged_attention.shared_prefix_attention(q, cache, _ints(lengths), prefix, **args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ROOMY[:3])
@pytest.mark.parametrize("new", [1, 4, 150])
def test_unassigned_table_entries(dtype, shape, new):
    """Table entries behind the last token or below every window are not looked at: no status, the same bits."""
    from strict_topk_overlap_b200 import _lib, paged_attention
    hq, hkv, d, block, page = shape
    length, window = 420, 200
    cache = _cache([length], hkv, d, block, page, dtype, 114, room=2 * block)
    q = _queries(new, hq, d, dtype, 115)
    lo = [p + 1 - window for p in range(length - new, length)]
    args = dict(token_offsets=None if new == 1 else _ints([0, new]), max_tokens=new, return_lse=True, kv_lo=_ints(lo))
    want = paged_attention.attention(q, cache, _ints([length]), **args)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.page_table[-(-length // page):] = -1
    cache.page_table[:lo[0] // page] = -1
    try:
        _lib.set_status_tensor(status)
        got = paged_attention.attention(q, cache, _ints([length]), **args)
    finally:
        _lib.set_status_tensor(None)
    assert int(status) == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 33, 16, 16), (3, 1, 5, 16, 8), (3, 3, 81, 32, 16), (1, 1, 1, 16, 16)])
@pytest.mark.parametrize("new,prefix", [(1, 0), (3, 0), (1, 64)])
def test_odd_heads_in_an_odd_number_of_parts(dtype, shape, new, prefix):
    """Partial states of an odd number of odd rows: what lies behind them in the workspace keeps its alignment."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    for length in (64 + 70, 190, 300):  # 3 and 5 parts of 64 keys
        cache = _cache([length], hkv, d, block, page, dtype, 116, shared=prefix)
        q = _queries(new, hq, d, dtype, 117)
        args = dict(token_offsets=None if new == 1 else _ints([0, new]), max_tokens=new, return_lse=True)
        if prefix:
            out, lse = paged_attention.shared_prefix_attention(q, cache, _ints([length]), prefix, **args)
        else:
            out, lse = paged_attention.attention(q, cache, _ints([length]), **args)
        _compare(q, cache, [length], [new], None, None, out, lse, 0.0, None, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", TILED)
@pytest.mark.parametrize("length,new", [(700, 40), (20000, 40), (20000, 300)])
@pytest.mark.parametrize("jump", [60.0, 80.0])
def test_scores_that_jump_under_large_values(dtype, shape, length, new, jump):
    """Scores that leave their frame far behind at the end of a part, times values that take the sum beyond FP32 there."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    cache = _cache([length], hkv, d, block, page, dtype, 118)
    at = _at(cache, 0, _span(0, length))
    cache.k_pages[at[0], :, at[1]] *= 0.25
    along = torch.where(_span(0, length) >= length - new - 60, jump, 0.0) * d ** 0.5 / 16
    cache.k_pages[at[0], :, at[1], 0] = along.to(dtype)[:, None].expand(-1, hkv)
    cache.v_pages *= 3e4 if dtype == torch.float16 else 1e7
    q = 0.25 * _queries(new, hq, d, dtype, 119)
    q[..., 0] = 16.0
    out, lse = paged_attention.attention(q, cache, _ints([length]), token_offsets=_ints([0, new]), max_tokens=new,
                                         return_lse=True)
    _compare(q, cache, [length], [new], None, None, out, lse, 0.0, None, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FORMS + [(24, 2, 128, 32, 16)])
@pytest.mark.parametrize("new,most", [([1, 1, 1], 1), ([2, 0, 1], 2), ([40, 3, 1], 40), ([150, 130, 0], 150)])
@pytest.mark.parametrize("pad", [1, 5, 300])
@pytest.mark.parametrize("prefix", [0, 96])
def test_padding_gets_zeros(dtype, shape, new, most, pad, prefix):
    """Tokens behind the last request's, as a padded graph has: zeros in the output, -inf in the log-sum-exp, no status;
    nothing else changes."""
    from strict_topk_overlap_b200 import _lib, paged_attention
    hq, hkv, d, block, page = shape
    prefix = prefix // block * block
    lengths = [prefix + max(1, n) + e for n, e in zip(new, (150, 20, 3))]
    t = sum(new)
    cache = _cache(lengths, hkv, d, block, page, dtype, 120, shared=prefix)
    q = _queries(t + pad, hq, d, dtype, 121)
    at = _ints(torch.tensor([0] + new).cumsum(0).tolist())
    args = dict(token_offsets=at, max_tokens=most, return_lse=True)
    ws = paged_attention.attention_workspace(cache, t + pad, hq, token_offsets=at, max_tokens=most, prefix=prefix)
    ws.fill_(255)
    stale = torch.full((t + pad, hq, d), float("nan"), dtype=dtype, device=DEV)  # what the output's memory held
    del stale
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    try:
        _lib.set_status_tensor(status)
        if prefix:
            out, lse = paged_attention.shared_prefix_attention(q, cache, _ints(lengths), prefix, workspace=ws, **args)
        else:
            out, lse = paged_attention.attention(q, cache, _ints(lengths), workspace=ws, **args)
    finally:
        _lib.set_status_tensor(None)
    assert int(status) == 0
    assert not bool(out[t:].any()) and bool((lse[t:] == float("-inf")).all())
    _compare(q[:t], cache, lengths, new, None, None, out[:t], lse[:t], 0.0, None, d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [1, 70])
def test_padding_is_not_appended(dtype, pad):
    """Padding's keys and values go nowhere, whatever its positions hold; its queries are turned by position 0."""
    from strict_topk_overlap_b200 import _lib, paged_append, rotary
    past, new, hq, hkv, d = [5, 40], [30, 2], 4, 2, 64
    g = torch.Generator(DEV).manual_seed(122)
    t = sum(new) + pad
    qkv = torch.randn((t, hq + 2 * hkv, d), generator=g, device=DEV).to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    turn = rotary.build_rotary(100, d)
    positions = torch.cat([_span(5, 35), _span(40, 42), torch.full((pad,), -9, device=DEV)]).to(torch.int32)
    caches = [paged_append.empty_paged_cache([64, 64], hkv, d, 32, 16, dtype=dtype,
                                             generator=torch.Generator().manual_seed(1)) for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full((t, hq, d), float("nan"), dtype=dtype, device=DEV)
    more = dict(token_offsets=_ints([0, 30, 32]), rotary=turn)
    try:
        _lib.set_status_tensor(status)
        paged_append.append_tokens(caches[0], k, v, _ints(past), q=q, q_out=out, positions=positions, **more)
    finally:
        _lib.set_status_tensor(None)
    n = sum(new)
    want = paged_append.append_tokens(caches[1], k[:n], v[:n], _ints(past), q=q[:n], positions=positions[:n].contiguous(), **more)
    assert int(status) == 0
    assert torch.equal(out[:n], want) and torch.equal(out[n:], q[n:])
    for name in ("k_pages", "v_pages", "lo", "hi"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))


@gpu
def test_offsets_that_do_not_begin_at_zero_are_reported():
    from strict_topk_overlap_b200 import _lib, paged_append, paged_attention
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = _cache([200, 300], 2, 64, 32, 16, torch.bfloat16, 123)
    try:
        _lib.set_status_tensor(status)
        for new in (3, 130):
            q = _queries(2 * new, 8, 64, torch.bfloat16, 124)
            paged_attention.attention(q, cache, _ints([200, 300]), token_offsets=_ints([1, new, 2 * new]), max_tokens=new)
            assert int(status) == 3
            status.zero_()
            kv = q[:, :2].contiguous()
            paged_append.append_tokens(cache, kv, kv, _ints([10, 20]), token_offsets=_ints([1, new, 2 * new]))
            assert int(status) == 3
            status.zero_()
    finally:
        _lib.set_status_tensor(None)


@gpu
def test_batches_of_different_sizes_from_several_threads():
    """Calls of one request and of thousands, from two threads at a time, do not disturb one another's launches."""
    import threading

    from strict_topk_overlap_b200 import paged_attention
    sizes, caches, wrong = (1, 15000), [], []
    for n in sizes:
        cache = _cache([16] * n, 1, 64, 16, 16, torch.bfloat16, 125)
        caches.append((cache, _queries(n, 2, 64, torch.bfloat16, 126), _ints([16] * n)))
    want = [paged_attention.attention(q, cache, at) for cache, q, at in caches]
    torch.cuda.synchronize()

    def work(i):
        cache, q, at = caches[i]
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(1500 if i == 0 else 300):
                    out = paged_attention.attention(q, cache, at)
                torch.cuda.current_stream().synchronize()
            if not torch.equal(out, want[i]):
                wrong.append("another result")
        except RuntimeError as e:
            wrong.append(str(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:2]


@gpu
@pytest.mark.parametrize("room", [0, 40])
def test_selection_over_a_cache_with_spare_room(room):
    """Blocks without tokens are never selected before blocks with some, and change nothing about those."""
    from strict_topk_overlap_b200 import paged, paged_append
    hq, hkv, d, block, page, filled = 8, 2, 128, 32, 16, [12, 30]
    g = torch.Generator(DEV).manual_seed(127)
    cache = paged_append.empty_paged_cache([(n + room) * block for n in filled], hkv, d, block, page,
                                           generator=torch.Generator().manual_seed(2))
    t = sum(filled) * block
    k, v = (torch.randn((t, hkv, d), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    paged_append.append_tokens(cache, k, v, _ints([0, 0]), token_offsets=_ints([0, filled[0] * block, t]))
    q = torch.randn((2 * hq, d), generator=g, device=DEV).to(torch.bfloat16)
    ids = paged.select_blocks(q, cache, 10).view(2, hq, 10)
    for r, n in enumerate(filled):
        first = sum(filled[:r]) * block
        keys = k[first:first + n * block].view(n, block, hkv, d).float()
        lo, hi = keys.amin(1), keys.amax(1)  # [n, hkv, d]
        x = q.view(2, hkv, hq // hkv, d)[r].double()
        score = torch.einsum("hgd,nhd->hgn", x.clamp(min=0), hi.double()) + torch.einsum("hgd,nhd->hgn", x.clamp(max=0), lo.double())
        want = score.reshape(hq, n).topk(10).indices
        assert torch.equal(ids[r].long().sort(-1).values, want.sort(-1).values)


def _strict(q, cache, lengths, new, lo, got, lse, softcap, slopes):
    """Against the definition in 64 bits, infinite and NaN outputs and log-sum-exps included: where the reference is
    not finite, the same value; elsewhere the tolerances of test_paged_attention.py."""
    dtype, d = q.dtype, q.shape[2]
    off, start = cache.block_offsets.tolist(), 0
    for r, (n, length) in enumerate(zip(new, lengths)):
        rows = slice(start, start + n)
        k, v = (O.gather(x, cache.page_table, off, cache.block_size, cache.page_size, r, length)
                for x in (cache.k_pages, cache.v_pages))
        pos = list(range(length - n, length))
        want, wlse, size, vmax = O.attention(q[rows], k, v, lo[rows] if lo else [0] * n, [p + 1 for p in pos], pos,
                                             scale=d ** -0.5, softcap=softcap, slopes=slopes)
        size = size.nan_to_num(0.0, 0.0)  # rows without a finite score are compared below
        ds = (d + 16) * 2.0 ** -24 * size + (1e-4 if dtype != torch.float32 else 0.0)
        u = UNIT[dtype]
        tol = u * want.abs() + ((0.0 if dtype == torch.float32 else u) + 2 * ds + 64 * 2.0 ** -24)[..., None] * vmax[..., None]
        out, ends = got[rows].double(), lse[rows].double()
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(ends.isnan(), wlse.isnan())
        odd = want.isinf()
        assert torch.equal(out[odd], want[odd]) and not bool(out[~odd].isinf().any())
        ok = want.isfinite()
        assert bool(((out - want).abs() <= tol)[ok].all())
        live = wlse.isfinite()
        assert bool(((ends - wlse).abs() <= ds + 64 * 2.0 ** -24 + 2.0 ** -22 * wlse.abs())[live].all())
        start += n


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FORMS)
@pytest.mark.parametrize("new", [1, 4, 200])
@pytest.mark.parametrize("scores", [dict(), dict(softcap=20.0), dict(biased=True)])
def test_seen_infinities(dtype, shape, new, scores):
    """Infinite values and infinite key elements at keys that some rows see: exactly the definition's infinities and
    NaN there, everything else as if nothing had happened."""
    from strict_topk_overlap_b200 import paged_attention
    hq, hkv, d, block, page = shape
    cache = _cache([300, 260], hkv, d, block, page, dtype, 128)
    q = _queries(2 * new, hq, d, dtype, 129)
    softcap = scores.get("softcap", 0.0)
    slopes = torch.full((hq,), 0.05, device=DEV) if scores.get("biased") else None
    pos = [p for length in (300, 260) for p in range(length - new, length)]
    lo = [p // 64 * 64 for p in pos]
    args = dict(token_offsets=None if new == 1 else _ints([0, new, 2 * new]), max_tokens=new, return_lse=True,
                softcap=softcap, slopes=slopes)
    for name, j, e, value in (("v_pages", 293, 5, float("inf")), ("v_pages", 259, 40, float("-inf")),
                              ("k_pages", 290, 3, float("inf")), ("k_pages", 257, d - 1, float("-inf"))):
        for low in (None, lo):
            pool = getattr(cache, name)
            held = pool.clone()
            for r in (0, 1):
                if j < (300, 260)[r]:
                    pg, slot = _at(cache, r, _span(j, j + 1))
                    pool[pg, :, slot, e] = value
            out, lse = paged_attention.attention(q, cache, _ints([300, 260]), kv_lo=None if low is None else _ints(low),
                                                 **args)
            _strict(q, cache, [300, 260], [new, new], low, out, lse, softcap, slopes)
            pool.copy_(held)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
def test_prefix_that_request_0_does_not_hold_is_reported(dtype, new):
    from strict_topk_overlap_b200 import _lib, paged_attention
    cache = _cache([50, 400], 2, 64, 32, 16, dtype, 130)
    q = _queries(2 * new, 8, 64, dtype, 131)
    args = dict(token_offsets=None if new == 1 else _ints([0, new, 2 * new]), max_tokens=new)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    try:
        _lib.set_status_tensor(status)
        paged_attention.shared_prefix_attention(q, cache, _ints([50, 400]), 64, **args)
        assert int(status) == 0
        paged_attention.shared_prefix_attention(q, cache, _ints([50, 400]), 96, **args)
        assert int(status) == 5
    finally:
        _lib.set_status_tensor(None)
