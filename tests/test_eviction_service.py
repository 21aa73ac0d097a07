"""The operators of a decode service within a budget, run together.

The appended keys and values of a sequence are known, so that what the service
kept can be checked token by token (moves are exact), and its last attention
against the definition over the kept tokens alone, within the bounds that
test_paged_attention.py derives."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import paged_dense as O
from test_paged_attention import UNIT

gpu = pytest.mark.gpu


def _service():
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_service.py"
    spec = importlib.util.spec_from_file_location("paged_service", path)
    service = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(service)
    return service


@gpu
@pytest.mark.parametrize("budget,slack", [(96, 32), (64, 1), (1000, 10)])
def test_service_within_a_budget(monkeypatch, budget, slack):
    """What is in the pool is what was appended at the places that are said to be kept: every key and value, the
    bounds of its blocks, and the last step's attention over it."""
    from strict_topk_overlap_b200 import paged_append, paged_attention
    service = _service()
    log, last = [], {}
    append, attend = paged_append.append_tokens, paged_attention.attention

    def logged(cache, k, v, lengths, **more):
        pool, table = cache.k_pages.clone(), cache.page_table
        q = append(cache, k, v, lengths, **more)
        log.append((k.clone(), v.clone(), lengths.clone(), more.get("token_offsets"), cache.k_pages, table))
        assert pool.shape == cache.k_pages.shape
        # The keys as they were stored (rotated), one per new token.
        off, page = cache.block_offsets.tolist(), cache.page_size
        start = more["token_offsets"].tolist() if more.get("token_offsets") is not None else list(range(len(off)))
        for r in range(cache.requests):
            n, at = start[r + 1] - start[r], int(lengths[r])
            kk = O.gather(cache.k_pages, table, off, cache.block_size, page, r, at + n)[:, at:]
            vv = O.gather(cache.v_pages, table, off, cache.block_size, page, r, at + n)[:, at:]
            keys.setdefault(r, []).append(kk.clone())
            values.setdefault(r, []).append(vv.clone())
        return q

    def kept(q, cache, lengths, **more):
        out = attend(q, cache, lengths, **more)
        last.update(q=q, out=out[0], lengths=lengths)
        return out

    keys, values = {}, {}
    monkeypatch.setattr(paged_append, "append_tokens", logged)
    monkeypatch.setattr(paged_attention, "attention", kept)
    cache, lengths, places, tokens = service.serve_within(budget, slack, say=lambda *_: None)
    assert tokens.shape == (80, 3) and bool(((tokens >= 0) & (tokens < 500)).all())
    off, block = cache.block_offsets.tolist(), cache.block_size
    for r in range(3):
        n = int(lengths[r])
        assert n <= budget + slack
        all_k, all_v = torch.cat(keys[r], 1), torch.cat(values[r], 1)
        k = O.gather(cache.k_pages, cache.page_table, off, block, cache.page_size, r, n)
        v = O.gather(cache.v_pages, cache.page_table, off, block, cache.page_size, r, n)
        at = places[r, :, :n]
        assert bool((at.diff(dim=-1) > 0).all())
        pick = at[..., None].expand(-1, -1, cache.dim)
        assert torch.equal(k, all_k.gather(1, pick)) and torch.equal(v, all_v.gather(1, pick))
        assert at[0, -1] == all_k.shape[1] - 1 and at[1, 0] == 0
        for j in range(-(-n // block)):
            part = k[:, j * block:(j + 1) * block].float()
            assert torch.equal(cache.lo[:, off[r] + j], part.amin(1)) and torch.equal(cache.hi[:, off[r] + j], part.amax(1))
        q, scale = last["q"][r:r + 1], cache.dim ** -0.5
        want, _, size, vmax = O.attention(q, k, v, [0], [n], [n - 1], scale=scale)
        ds = (cache.dim + 16) * 2.0 ** -24 * size + 1e-4
        u = UNIT[torch.bfloat16]
        tol = u * want.abs() + (u + 2 * ds + 64 * 2.0 ** -24)[..., None] * vmax[..., None]
        assert bool(((last["out"][r:r + 1].double() - want).abs() <= tol).all())
