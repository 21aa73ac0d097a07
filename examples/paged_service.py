"""A small decode service over a paged cache, for one layer's attention: the
prompts' tokens enter the page pool rotated, attend over it, and are followed
by a few decode steps, each one an append, a dense attention and a strict Top-K
selection whose block-sparse attention reads the same pages. Behind a system
prompt that all requests share, its pages are stored and attended once.

    python examples/paged_service.py [--requests 8] [--system 1024] [--steps 4]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from strict_topk_overlap_b200 import paged, paged_append, paged_attention, rotary  # noqa: E402

HQ, HKV, D, BLOCK, PAGE, TOPK = 32, 8, 128, 32, 16, 8


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def projections(tokens, gen):
    """A layer's q, k, v of some tokens, as slices of one projection's output."""
    qkv = torch.randn((tokens, HQ + 2 * HKV, D), generator=gen, device="cuda").to(torch.bfloat16)
    return qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]


def shared_cache(cache, requests, system):
    """The cache with every request's table beginning with request 0's system blocks."""
    ppb, blocks = BLOCK // PAGE, system // BLOCK
    table, start = cache.page_table.clone(), cache.block_offsets.tolist()
    for r in range(1, requests):
        table[start[r] * ppb:(start[r] + blocks) * ppb] = table[:blocks * ppb]
        cache.lo[:, start[r]:start[r] + blocks] = cache.lo[:, :blocks]
        cache.hi[:, start[r]:start[r] + blocks] = cache.hi[:, :blocks]
    cache.page_table = table


def serve(requests=8, system=1024, steps=4, seed=0, say=print):
    """Returns the largest difference between the shared and the plain attention of the steps."""
    gen = torch.Generator("cuda").manual_seed(seed)
    own = [BLOCK * (1 + r % 3) - steps for r in range(requests)]  # the last step fills the requests' blocks
    cache = paged_append.empty_paged_cache([system + n + steps for n in own], HKV, D, BLOCK, PAGE,
                                           generator=torch.Generator().manual_seed(seed))
    turn = rotary.build_rotary(system + max(own) + steps, D)

    # The system prompt, once, into request 0's blocks; the others' tables then name the same pages.
    q, k, v = projections(system, gen)
    one = paged.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table, cache.block_offsets[:2].contiguous(),
                             cache.lo, cache.hi, BLOCK, PAGE, cache.max_blocks)
    q = paged_append.append_tokens(one, k, v, ints([0]), token_offsets=ints([0, system]), q=q, rotary=turn)
    paged_attention.attention(q, one, ints([system]), token_offsets=ints([0, system]))
    shared_cache(cache, requests, system)

    # The requests' own prompts, packed.
    offsets = ints([sum(own[:r]) for r in range(requests + 1)])
    lengths = ints([system] * requests)
    q, k, v = projections(sum(own), gen)
    q = paged_append.append_tokens(cache, k, v, lengths, token_offsets=offsets, q=q, rotary=turn)
    lengths += ints(own)
    out = paged_attention.shared_prefix_attention(q, cache, lengths, system, token_offsets=offsets, max_tokens=max(own))
    say(f"prompts: {sum(own)} tokens behind {system} shared ones -> {tuple(out.shape)}")

    worst = 0.0
    for step in range(steps):
        q, k, v = projections(requests, gen)
        q = paged_append.append_tokens(cache, k, v, lengths, q=q, rotary=turn)
        lengths += 1
        out = paged_attention.shared_prefix_attention(q, cache, lengths, system)
        plain = paged_attention.attention(q, cache, lengths)
        worst = max(worst, float((out.float() - plain.float()).abs().max()))
    # All blocks are full now: the same pages and bounds serve the block-sparse path.
    rows = q.reshape(requests * HQ, D)
    topk = min(TOPK, (system + min(own) + steps) // BLOCK)
    selected = paged.select_blocks(rows, cache, topk)
    sparse = paged.exact(rows, cache, selected)
    say(f"{steps} steps: shared and plain attention differ by {worst:.1e}; "
        f"block-sparse attention of {topk} blocks -> {tuple(sparse.shape)}")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--system", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=4)
    a = ap.parse_args()
    serve(a.requests, a.system, a.steps)
