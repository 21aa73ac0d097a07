"""A small decode service over a paged cache, for one layer's attention: the
prompts' tokens enter the page pool rotated, attend over it, and are followed
by a few decode steps, each one an append, a dense attention and a strict Top-K
selection whose block-sparse attention reads the same pages. Behind a system
prompt that all requests share, its pages are stored and attended once.
Requests that outgrow their share of the pool are cut back to the tokens that
are attended most, and tokens are drawn from a head's logits on the way
(``serve_within``).

    python examples/paged_service.py [--requests 8] [--system 1024] [--steps 4] [--budget 96]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from strict_topk_overlap_b200 import paged, paged_append, paged_attention, paged_eviction, rotary, sampling  # noqa: E402

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


def serve_within(budget=96, slack=32, prompts=(200, 40, 130), steps=80, sinks=4, recent=16, vocabulary=500, seed=0, say=print):
    """Decodes with at most budget + slack tokens of a request in the pool: whenever that many are there, what was
    attended least is evicted down to the budget. Each step's token is drawn from the logits of a random head and fed
    back as the next step's embedding. Returns the cache, its lengths, the places in the sequence of the cached tokens
    of each KV head, and the drawn tokens."""
    gen = torch.Generator("cuda").manual_seed(seed)
    requests = len(prompts)
    room = max(max(prompts), budget + slack)
    cache = paged_append.empty_paged_cache([room] * requests, HKV, D, BLOCK, PAGE, generator=torch.Generator().manual_seed(seed))
    turn = rotary.build_rotary(max(prompts) + steps, D)
    weights = paged_eviction.empty_weights(cache)
    embeddings = torch.randn((vocabulary, (HQ + 2 * HKV) * D), generator=gen, device="cuda").to(torch.bfloat16)
    head = torch.randn((HQ * D, vocabulary), generator=gen, device="cuda").to(torch.bfloat16)

    # The prompts; their last tokens' attention is the first word on what is kept.
    offsets = ints([sum(prompts[:r]) for r in range(requests + 1)])
    q, k, v = projections(sum(prompts), gen)
    q = paged_append.append_tokens(cache, k, v, ints([0] * requests), token_offsets=offsets, q=q, rotary=turn)
    lengths = ints(prompts)
    out, lse = paged_attention.attention(q, cache, lengths, token_offsets=offsets, max_tokens=max(prompts), return_lse=True)
    paged_eviction.accumulate_weights(weights, q, cache, lengths, lse, token_offsets=offsets, max_tokens=max(prompts))
    places = torch.arange(room, device="cuda").expand(requests, HKV, room)
    out = out[offsets[1:].long() - 1]
    seen, tokens = list(prompts), []
    held = list(prompts)  # lengths, as the host knows them
    for _ in range(steps):
        if max(held) >= budget + slack:
            lengths, kept = paged_eviction.evict(cache, weights, lengths, budget, first=sinks, last=recent)
            held = [min(n, budget) for n in held]
            moved = torch.gather(places, 2, kept.long().clamp(min=0))
            places = torch.cat((torch.where(kept < 0, 0, moved), places[..., budget:]), -1)
        logits = out.flatten(1) @ head
        tokens.append(sampling.sample(logits, torch.rand((requests,), generator=gen, device="cuda"), temperature=0.8, top_k=40,
                                      top_p=0.95))
        qkv = embeddings[tokens[-1].long()].view(requests, HQ + 2 * HKV, D)
        # The kept keys stay rotated as they were: a new token has its place in the sequence, not the one in the pool.
        q = paged_append.append_tokens(cache, qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], lengths, q=qkv[:, :HQ], rotary=turn,
                                       positions=ints(seen))
        places = places.scatter(2, lengths.long()[:, None, None].expand(requests, HKV, 1),
                                ints(seen).long()[:, None, None].expand(requests, HKV, 1))
        lengths = lengths + 1
        seen, held = [n + 1 for n in seen], [n + 1 for n in held]
        out, lse = paged_attention.attention(q, cache, lengths, return_lse=True)
        paged_eviction.accumulate_weights(weights, q, cache, lengths, lse)
    say(f"{steps} steps within {budget} + {slack} tokens a request: {held} of {seen} tokens are kept")
    return cache, lengths, places, torch.stack(tokens)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--system", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--budget", type=int, default=96)
    a = ap.parse_args()
    serve(a.requests, a.system, a.steps)
    serve_within(a.budget)
