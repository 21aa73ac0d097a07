"""Appending rotated tokens to a paged cache against its definition in 64 bits.

Stored values are the FP32 formula rounded once: with u the type's rounding
unit (2^-8, 2^-11, 2^-24 relative for bf16, f16, f32) a value x = a c - b s is
off by at most u |x| for the last rounding, 3 * 2^-24 (|a c| + |b s|) for the
two products and the sum, and 2^-25 absolute for f16's subnormals. The bounds
are compared bit for bit with the minimum and maximum of the stored keys."""
from __future__ import annotations

import pytest
import torch

from oracle import paged_dense as O

gpu = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _inputs(past, new, hq, hkv, d, block, page, dtype, seed, bounds=True):
    """A cache with room for the requests' tokens, and the new tokens' q, k, v as slices of one tensor."""
    from strict_topk_overlap_b200 import paged_append
    g = torch.Generator().manual_seed(seed)
    cache = paged_append.empty_paged_cache([max(1, p + n) for p, n in zip(past, new)], hkv, d, block, page,
                                           dtype=dtype, bounds=bounds, generator=g, device=DEV)
    t = sum(new)
    qkv = torch.randn((t, hq + 2 * hkv, d), generator=g).to(dtype).to(DEV)
    offsets = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=DEV)
    return cache, qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], offsets


def _near(got, want, size, dtype):
    tol = UNIT[dtype] * want.abs() + 3 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    worst = ((got.double() - want).abs() - tol).max()
    assert float(worst) <= 0, float(worst)


def _check(cache, q, k, v, q_out, past, new, offsets, rotary, places):
    """places [T, pairs]: table rows."""
    off = cache.block_offsets.tolist()
    dtype = k.dtype
    for r, (p, n) in enumerate(zip(past, new)):
        rows = slice(int(offsets[r]), int(offsets[r + 1]))
        args = (rotary.cos, rotary.sin, rotary.interleaved, places[rows])
        sizes = (rotary.cos.abs(), rotary.sin.abs())
        for x, y in ((q, q_out), (k, None)):
            if x is None:
                continue
            got = y[rows] if y is not None else O.gather(cache.k_pages, cache.page_table, off, cache.block_size,
                                                         cache.page_size, r, p + n)[:, p:].transpose(0, 1)
            want = O.rotate(x[rows], *args)
            pairs = rotary.cos.shape[1]
            size = want.abs()
            i = torch.arange(pairs, device=DEV)
            a, b = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + pairs)
            c = sizes[0].double().gather(0, places[rows])[:, None]
            s = sizes[1].double().gather(0, places[rows])[:, None]
            xa = x[rows].double().abs()
            size[..., a] = xa[..., a] * c + xa[..., b] * s
            size[..., b] = xa[..., b] * c + xa[..., a] * s
            if n:
                _near(got, want, size, dtype)
        got_v = O.gather(cache.v_pages, cache.page_table, off, cache.block_size, cache.page_size, r, p + n)[:, p:]
        assert torch.equal(got_v.transpose(0, 1), v[rows])
        keys = O.gather(cache.k_pages, cache.page_table, off, cache.block_size, cache.page_size, r, p + n).float()
        if cache.total_blocks and p + n:
            for j in range((p + n - 1) // cache.block_size + 1):
                part = keys[:, j * cache.block_size:(j + 1) * cache.block_size]
                assert torch.equal(cache.lo[:, off[r] + j], part.amin(1)), (r, j)
                assert torch.equal(cache.hi[:, off[r] + j], part.amax(1)), (r, j)


SHAPES = [  # hq, hkv, d, rotated dims, block, page
    (8, 2, 128, 128, 32, 16), (4, 4, 64, 32, 64, 16), (6, 2, 80, 80, 16, 8), (3, 1, 48, 20, 24, 3), (2, 1, 65, 6, 4, 1),
    (2, 2, 256, 256, 32, 32), (1, 1, 576, 64, 8, 8)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_ragged(dtype, shape, interleaved):
    from strict_topk_overlap_b200 import paged_append, rotary
    hq, hkv, d, rot, block, page = shape
    table = rotary.build_rotary(300, rot, interleaved=interleaved, device=DEV)
    steps = [[0, 5, 1, 33, 130], [70, 0, 1, 2, 63], [1, 1, 1, 1, 1]]  # appended one after the other
    total = [sum(x) for x in zip(*steps)]
    past = [0] * 5
    cache = None
    for s, new in enumerate(steps):
        fresh, q, k, v, offsets = _inputs([0] * 5, total if s == 0 else new, hq, hkv, d, block, page, dtype, 10 + s)
        if s == 0:
            cache = fresh
            q, k, v = (x[:sum(new)] for x in (q, k, v))
            offsets = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=DEV)
        lengths = torch.tensor(past, dtype=torch.int32, device=DEV)
        single = all(n == 1 for n in new)
        out = paged_append.append_tokens(cache, k, v, lengths, token_offsets=None if single else offsets, q=q,
                                         rotary=table)
        at = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(DEV)
        _check(cache, q, k, v, out, past, new, offsets, table, at[:, None].expand(-1, rot // 2))
        past = [p + n for p, n in zip(past, new)]


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_several_axes(interleaved, dtype):
    from strict_topk_overlap_b200 import paged_append, rotary
    table = rotary.build_rotary(100, 96, interleaved=interleaved, sections=(8, 20, 20), device=DEV)
    new = [37, 64]
    cache, q, k, v, offsets = _inputs([0, 0], new, 4, 2, 128, 32, 16, dtype, 5)
    positions = torch.randint(0, 100, (3, sum(new)), dtype=torch.int32, generator=torch.Generator().manual_seed(2)).to(DEV)
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    out = paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets, q=q, rotary=table,
                                     positions=positions)
    places = positions[table.axis.long()].t().long()
    _check(cache, q, k, v, out, [0, 0], new, offsets, table, places)
    # One axis of given positions.
    line = rotary.build_rotary(100, 96, interleaved=interleaved, device=DEV)
    out = paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets, q=q, rotary=line,
                                     positions=positions[0].contiguous())
    _check(cache, q, k, v, out, [0, 0], new, offsets, line, positions[0].long()[:, None].expand(-1, 48))


@gpu
def test_append_strides_in_place_and_without_rotation():
    from strict_topk_overlap_b200 import paged_append, rotary
    new = [50]
    cache, q, k, v, offsets = _inputs([0], new, 4, 2, 64, 32, 16, torch.bfloat16, 9)
    lengths = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets)
    assert torch.equal(O.gather(cache.k_pages, cache.page_table, [0, 2], 32, 16, 0, 50).transpose(0, 1), k)
    # Rows that start at an odd element, and head-major strides.
    table = rotary.build_rotary(64, 64, device=DEV)
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape)
    odd.copy_(k)
    turned = v.transpose(0, 1).contiguous().transpose(0, 1)
    mine = q.contiguous()
    out = paged_append.append_tokens(cache, odd, turned, lengths, token_offsets=offsets, q=mine.clone(), rotary=table)
    at = torch.arange(50, device=DEV)[:, None].expand(-1, 32)
    _check(cache, mine, k, v, out, [0], new, offsets, table, at)
    same = mine.clone()
    assert paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets, q=same, rotary=table,
                                      q_out=same) is same
    assert torch.equal(same, out)


@gpu
def test_append_nan_keys_and_no_bounds():
    from strict_topk_overlap_b200 import paged_append
    cache, q, k, v, offsets = _inputs([0], [40], 2, 2, 64, 32, 16, torch.bfloat16, 3)
    k = k.clone()
    k[3, 0, 5] = float("nan")
    k[4, 1, 7] = float("inf")
    lengths = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets)
    want = k[:32].float().transpose(0, 1)
    assert torch.equal(cache.lo[:, 0].isnan(), want.amin(1).isnan())
    assert torch.equal(cache.hi[:, 0].nan_to_num(7e9), want.amax(1).nan_to_num(7e9))
    bare, _, _, _, _ = _inputs([0], [40], 2, 2, 64, 32, 16, torch.bfloat16, 3, bounds=False)
    paged_append.append_tokens(bare, k, v, lengths, token_offsets=offsets)
    assert torch.equal(bare.v_pages[bare.page_table[0].long()], cache.v_pages[cache.page_table[0].long()])


@gpu
def test_append_feeds_block_selection():
    """The bounds left by the append select the blocks that bounds rebuilt from the keys select."""
    from strict_topk_overlap_b200 import paged, paged_append, rotary
    new = [32 * 9, 32 * 5]
    cache, q, k, v, offsets = _inputs([0, 0], new, 8, 2, 128, 32, 16, torch.bfloat16, 4)
    table = rotary.build_rotary(400, 128, device=DEV)
    paged_append.append_tokens(cache, k, v, torch.zeros(2, dtype=torch.int32, device=DEV), token_offsets=offsets,
                               rotary=table)
    query = torch.randn(16, 128, device=DEV).to(torch.bfloat16)
    got = paged.select_blocks(query, cache, 4)
    off = cache.block_offsets.tolist()
    ks = [O.gather(cache.k_pages, cache.page_table, off, 32, 16, r, n).view(2, -1, 32, 128) for r, n in enumerate(new)]
    again = paged.build_paged_cache(ks, ks, 16, device=torch.device(DEV))
    assert torch.equal(got, paged.select_blocks(query, again, 4))


@gpu
def test_append_reports_bad_data():
    from strict_topk_overlap_b200 import _lib, paged_append, rotary
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(1, dtype=torch.int32, device=DEV)
    try:
        _lib.set_status_tensor(status)
        # Tokens beyond the request's two blocks are dropped, the others written.
        cache, q, k, v, offsets = _inputs([0], [70], 2, 2, 64, 32, 16, torch.bfloat16, 3)
        small, _, _, _, _ = _inputs([0], [64], 2, 2, 64, 32, 16, torch.bfloat16, 3)
        paged_append.append_tokens(small, k, v, lengths, token_offsets=offsets)
        assert int(status) == 5
        assert torch.equal(O.gather(small.k_pages, small.page_table, [0, 2], 32, 16, 0, 64).transpose(0, 1), k[:64])
        status.zero_()
        paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets, q=q,
                                   rotary=rotary.build_rotary(50, 64, device=DEV))
        assert int(status) == 4
        status.zero_()
        cache.page_table[1] = cache.k_pages.shape[0]
        paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets)
        assert int(status) == 2
        status.zero_()
        paged_append.append_tokens(small, k[:64], v[:64], lengths - 1,
                                   token_offsets=torch.tensor([0, 64], dtype=torch.int32, device=DEV))
        assert int(status) == 5
    finally:
        _lib.set_status_tensor(None)


@gpu
def test_append_refusals():
    from strict_topk_overlap_b200 import paged_append, rotary
    cache, q, k, v, offsets = _inputs([0, 0], [3, 4], 4, 2, 64, 32, 16, torch.bfloat16, 3)
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    table = rotary.build_rotary(50, 64, device=DEV)
    ok = dict(token_offsets=offsets, q=q, rotary=table)
    call = paged_append.append_tokens
    for bad in (dict(k=k[:, :1]), dict(v=v[:3]), dict(k=k.float()), dict(k=k.transpose(1, 2)), dict(lengths=lengths.long()),
                dict(lengths=lengths[:1]), dict(token_offsets=offsets[:2]), dict(token_offsets=None),
                dict(q=q[:, :3]), dict(q=q[:2]), dict(q_out=q), dict(positions=offsets),
                dict(positions=torch.zeros((3, 7), dtype=torch.int32, device=DEV)),
                dict(rotary=rotary.Rotary(table.cos.half(), table.sin)),
                dict(rotary=rotary.Rotary(table.cos, table.sin, axis=torch.zeros(32, dtype=torch.uint8, device=DEV))),
                dict(rotary=None, positions=torch.zeros(7, dtype=torch.int32, device=DEV))):
        args = dict(k=k, v=v, lengths=lengths, **ok)
        args.update(bad)
        with pytest.raises(ValueError):
            call(cache, args.pop("k"), args.pop("v"), args.pop("lengths"), **args)
    with pytest.raises(RuntimeError, match="rotary"):
        call(cache, k, v, lengths, token_offsets=offsets, rotary=rotary.build_rotary(50, 128, device=DEV))


def test_tables():
    """CPU: the table's values and its refusals."""
    from strict_topk_overlap_b200 import paged_append, rotary
    t = rotary.build_rotary(7, 6, base=100.0, sections=(1, 0, 2), device="cpu")
    want = torch.arange(7, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(3, dtype=torch.float64) / 3)
    assert torch.equal(t.cos, want.cos().float()) and torch.equal(t.sin, want.sin().float())
    assert t.axis.tolist() == [0, 2, 2] and t.axis.dtype == torch.uint8
    for bad in (dict(max_position=0, dim=4), dict(max_position=4, dim=5), dict(max_position=4, dim=8, sections=(1, 2))):
        with pytest.raises(ValueError):
            rotary.build_rotary(**bad, device="cpu")
    for bad in (([], 32, 16), ([0], 32, 16), ([4], 32, 12)):
        with pytest.raises(ValueError):
            paged_append.empty_paged_cache(bad[0], 2, 64, bad[1], bad[2], device="cpu")
    cache = paged_append.empty_paged_cache([33, 1], 2, 64, 32, 16, device="cpu")
    assert cache.block_offsets.tolist() == [0, 2, 3] and sorted(cache.page_table.tolist()) == list(range(6))
