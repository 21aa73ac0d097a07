"""Cases for keeping a decode service's cache small and for what follows its
last layer: the attention weight that each cached key receives, eviction of
the tokens that received least, and sampling of the next tokens from given
random numbers.

``run`` computes each operator in elementary torch operations (FP32, rounded
once at the end; sampling in FP64, whose sums decide between neighbouring
tokens), or, with ``own`` set, through the package's entry points on the same
inputs. Page pools are [pages, Hkv, page, D], block g of the batch is made of
the pages page_table[g * block / page + i], and request r owns the blocks
block_offsets[r] .. block_offsets[r + 1]. Accumulated weights are FP32
[Hkv, blocks, block], one per KV head and token slot of a block.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EMPTY = 1e30  # lo, and minus hi, of a block without tokens


# ------------------------------------------------------------------ the cases

def _weigh(name, dtype, hq, hkv, d, requests, past, new, *, block=32, page=16, window=0, cap=0.0, slopes=False, seed=7):
    case = {"op": "weigh", "dtype": dtype, "hq": hq, "hkv": hkv, "d": d, "block": block, "page": page,
            "requests": requests, "past_min": past[0], "past_max": past[1], "new_min": new[0], "new_max": new[1],
            "window": window, "cap": cap, "slopes": slopes, "shape_seed": seed}
    return {"name": name, **case} if name else case


def _evict(name, dtype, hkv, d, requests, held, keep, first, last, *, block=32, page=16, seed=7):
    case = {"op": "evict", "dtype": dtype, "hkv": hkv, "d": d, "block": block, "page": page, "requests": requests,
            "held_min": held[0], "held_max": held[1], "keep": keep, "first": first, "last": last, "shape_seed": seed}
    return {"name": name, **case} if name else case


def _sample(name, dtype, rows, vocabulary, temperature, top_k, top_p, min_p, mixed, spread=2.5):
    case = {"op": "sample", "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "spread": spread}
    return {"name": name, **case} if name else case


def listed():
    return [
        # A decode step of one request of a small model: latency is what counts.
        _weigh("weigh-step-1", "bf16", 8, 2, 128, 1, (4095, 4095), (1, 1)),
        # A decode step of 64 requests of 8 K to 32 K tokens.
        _weigh("weigh-step-64", "bf16", 16, 8, 128, 64, (8191, 32767), (1, 1)),
        # The smallest type that has no tensor cores: a step of a few requests in FP32.
        _weigh("weigh-step-f32", "f32", 32, 8, 128, 5, (700, 9000), (1, 1)),
        # What the last 64 tokens of long prompts attend to, which decides what of the prompts is kept.
        _weigh("weigh-last-64", "bf16", 32, 8, 128, 4, (17000, 32000), (64, 64)),
        # All tokens of three prompts, their scores capped.
        _weigh("weigh-prompts", "bf16", 16, 8, 128, 3, (0, 0), (1500, 8192), cap=50.0),
        # A packed batch of prompts in a sliding window, biased by distance, heads of 64 dims.
        _weigh("weigh-window", "f16", 32, 8, 64, 6, (0, 900), (100, 5000), window=1024, slopes=True),
        # One request is cut back to its budget, as it is every few steps.
        _evict("evict-1", "bf16", 2, 128, 1, (4128, 4128), 4096, 4, 64),
        # Long prompts are cut to 2 K tokens each, the shortest of them have less.
        _evict("evict-prompts", "bf16", 8, 128, 16, (1500, 32000), 2048, 16, 128),
        # A few long requests keep 16 K tokens: moving the cache is the work.
        _evict("evict-long", "f16", 8, 128, 6, (20000, 60000), 16384, 64, 1000),
        # The next token of one request.
        _sample("sample-1", "f32", 1, 32001, 0.8, 50, 0.9, 0.0, False),
        # 64 requests, a large vocabulary, no bound on the number of tokens.
        _sample("sample-64", "f32", 64, 131072, 1.0, 0, 0.95, 0.0, False),
        # A large batch whose requests ask for different things, greedy ones among them; 16-bit logits, many equal.
        _sample("sample-256", "bf16", 256, 50257, 0.7, 40, 0.9, 0.05, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv = rng.choice(((32, 8), (16, 8), (8, 2), (96, 8), (8, 8)))
    d, page, block = rng.choice((64, 128)), rng.choice((16, 32)), rng.choice((32, 64))
    seed = rng.randrange(1 << 20)
    op = rng.choice(("step", "some", "prompt", "evict", "sample"))
    more = {"block": block, "page": page, "seed": seed}
    while True:
        if op == "step":
            dtype, requests, top = rng.choice(("bf16", "f16", "f32")), _log(rng, 1, 64), _log(rng, 64, 65536)
            case = _weigh(None, dtype, hq, hkv, d, requests, (top // 4, top), (1, 1),
                          window=rng.choice((0, 0, _log(rng, 16, top))), cap=rng.choice((0.0, 50.0)),
                          slopes=rng.random() < 0.3, **more)
            if requests * top * hkv * d * (2 if dtype == "f32" else 1) <= 64 * 20000 * 8 * 128:
                return case
        elif op == "some":  # drafts, or the last tokens of prompts
            requests, top, new = _log(rng, 1, 16), _log(rng, 64, 32000), _log(rng, 2, 128)
            case = _weigh(None, rng.choice(("bf16", "f16")), hq, hkv, d, requests, (top // 3, top), (max(1, new // 2), new),
                          window=rng.choice((0, 0, _log(rng, 16, top))), cap=rng.choice((0.0, 30.0)),
                          slopes=rng.random() < 0.3, **more)
            if requests * top * new * hq <= 4 * 32000 * 64 * 32:
                return case
        elif op == "prompt":
            requests, top = _log(rng, 1, 8), _log(rng, 32, 8000)
            past = rng.choice((0, 0, _log(rng, 32, 16000)))
            case = _weigh(None, rng.choice(("bf16", "f16")), hq, hkv, d, requests, (past // 2, past), (1, top),
                          window=rng.choice((0, 0, _log(rng, 16, top + past))), cap=rng.choice((0.0, 30.0, 50.0)),
                          slopes=rng.random() < 0.3, **more)
            if requests * hq * top * (top + past) * d <= 3 * 16 * 8192 * 8192 * 128:
                return case
        elif op == "evict":
            requests, top = _log(rng, 1, 64), _log(rng, 64, 60000)
            keep = max(8, int(top * rng.uniform(0.05, 0.9)))
            case = _evict(None, rng.choice(("bf16", "f16", "f32")), hkv, d, requests, (top // 3, top), keep,
                          rng.choice((0, 4, keep // 8)), rng.choice((0, 1, keep // 3)), **more)
            if requests * top * hkv * d * (2 if case["dtype"] == "f32" else 1) <= 6 * 60000 * 8 * 128:
                return case
        else:
            rows, vocabulary = _log(rng, 1, 256), _log(rng, 1000, 200000)
            case = _sample(None, rng.choice(("bf16", "f16", "f32")), rows, vocabulary, rng.choice((0.0, 0.6, 1.0, 1.3)),
                           rng.choice((0, 0, 1, 20, 1000)), rng.choice((1.0, 0.5, 0.9, 0.99)),
                           rng.choice((0.0, 0.0, 0.02)), rng.random() < 0.5, rng.choice((0.5, 2.5, 6.0)))
            if rows * vocabulary <= 256 * 50257:
                return case


def _lengths(case):
    """Tokens in the cache before the call, and new ones, per request."""
    rng = random.Random(case["shape_seed"])
    past = [rng.randint(case["past_min"], case["past_max"]) for _ in range(case["requests"])]
    return past, [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["requests"])]


def _held(case):
    rng = random.Random(case["shape_seed"])
    return [rng.randint(case["held_min"], case["held_max"]) for _ in range(case["requests"])]


def _cumulative(counts):
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return total


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocabulary"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2), "flops": 4 * n}
    hkv, d, size = case["hkv"], case["d"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "evict":
        held, keep = _held(case), case["keep"]
        moved = sum(keep - case["first"] for n in held if n > keep)
        slots = sum(-(-n // case["block"]) for n in held) * case["block"]
        blocks = sum(-(-keep // case["block"]) for n in held if n > keep)
        rest = 4 * hkv * (sum(held) + slots + len(held) * keep) + 8 * hkv * d * blocks
        return {"bytes": 4 * moved * hkv * d * size + rest, "flops": 2 * moved * hkv * d}
    past, new = _lengths(case)
    hq, w = case["hq"], case["window"]
    pairs = seen = 0
    for p, n in zip(past, new):
        full = lambda m: m * (m + 1) // 2  # noqa: E731
        pairs += full(p + n) - full(p)
        if w:
            pairs -= full(max(0, p + n - w)) - full(max(0, p - w))
        seen += p + n - (max(0, p + 1 - w) if w else 0)
    return {"bytes": sum(new) * hq * (d * size + 4) + seen * hkv * (d * size + 8), "flops": 2 * pairs * hq * d}


# ------------------------------------------------------------------ inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _cache(case, gen, lengths):
    b, page, hkv, d = case["block"], case["page"], case["hkv"], case["d"]
    blocks = [-(-n // b) for n in lengths]
    pages = sum(blocks) * (b // page)
    shape = (pages, hkv, page, d)
    dtype = DTYPES[case["dtype"]]
    k = torch.randn(shape, generator=gen, device=DEV, dtype=dtype)
    k += 0.5 * torch.randn((pages, hkv, 1, d), generator=gen, device=DEV, dtype=dtype)  # neighbouring tokens are alike
    none = torch.empty((hkv, 0, d), device=DEV)  # a cache that no block selection reads keeps no bounds
    return {"case": case, "k_pages": k, "v_pages": torch.randn(shape, generator=gen, device=DEV, dtype=dtype),
            "table": torch.randperm(pages, generator=gen, device=DEV).to(torch.int32),  # as an allocator leaves them
            "block_offsets": _ints(_cumulative(blocks)), "max_blocks": max(blocks), "blocks": sum(blocks),
            "lo": none, "hi": none}


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, gen)
    if case["op"] == "evict":
        held = _held(case)
        s = _cache(case, gen, held)
        b, ppb, page, hkv = case["block"], case["block"] // case["page"], case["page"], case["hkv"]
        s["lengths"] = _ints(held)
        place = torch.cat([torch.arange(-(-n // b) * b) for n in held]).to(DEV)
        end = torch.cat([torch.full((-(-n // b) * b,), n) for n in held]).to(DEV)
        live = place < end
        # A few tokens receive most of the weight, the newest little, some none at all.
        w = torch.exp(2 * torch.randn((hkv, place.numel()), generator=gen, device=DEV))
        w *= ((end - place) / end).sqrt() * (torch.rand(w.shape, generator=gen, device=DEV) > 0.1)
        s["weights"] = torch.where(live, w, 0.0).view(hkv, s["blocks"], b)
        s["weights_out"] = torch.empty_like(s["weights"])
        cached = s["k_pages"][s["table"].long()].view(-1, ppb, hkv, page, case["d"])
        filled = live.view(-1, ppb, 1, page, 1)
        s["lo"] = torch.where(filled, cached.float(), math.inf).amin((1, 3)).transpose(0, 1).contiguous()
        s["hi"] = torch.where(filled, cached.float(), -math.inf).amax((1, 3)).transpose(0, 1).contiguous()
        return s
    past, new = _lengths(case)
    t, hq = sum(new), case["hq"]
    s = _cache(case, gen, [p + n for p, n in zip(past, new)])
    s |= {"max_new": max(new), "lengths": _ints([p + n for p, n in zip(past, new)]),
          "token_offsets": None if max(new) == 1 else _ints(_cumulative(new)), "kv_lo": None, "slopes": None}
    s["q"] = torch.randn((t, hq, case["d"]), generator=gen, device=DEV, dtype=DTYPES[case["dtype"]])
    if case["window"]:
        s["kv_lo"] = _ints([max(0, i + 1 - case["window"]) for p, n in zip(past, new) for i in range(p, p + n)])
    if case["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV)
    # What earlier steps have added, and the log-sum-exps that the attention of these tokens returned.
    s["weights"] = torch.rand((case["hkv"], s["blocks"], case["block"]), generator=gen, device=DEV) * (0.001 if max(past) else 0.0)
    s["lse"] = torch.empty((t, hq), device=DEV)
    for r, rows, h, x in _parts(s, past, new, torch.float32):
        s["lse"][rows, h] = torch.logsumexp(x, -1).t()
    return s


def _parts(s, past, new, kind):
    """The scores of the definition in pieces: (request, rows, heads, [G, rows, keys]) of one KV head and at most 2,048 rows."""
    case = s["case"]
    hkv, d, g = case["hkv"], case["d"], case["hq"] // case["hkv"]
    ppb, offsets, start = case["block"] // case["page"], s["block_offsets"].tolist(), _cumulative(new)
    for r, (p, n) in enumerate(zip(past, new)):
        pages = s["table"].long()[offsets[r] * ppb:offsets[r + 1] * ppb]
        key = torch.arange(p + n, device=DEV)
        for h in range(hkv):
            heads = slice(h * g, (h + 1) * g)
            k = s["k_pages"][pages, h].reshape(-1, d)[:p + n].to(kind)
            for at in range(0, n, 2048):
                place = torch.arange(p + at, p + min(n, at + 2048), device=DEV)[:, None]
                rows = slice(start[r] + at, start[r] + min(n, at + 2048))
                x = s["q"][rows, heads].to(kind).transpose(0, 1) @ k.t() / math.sqrt(d)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][heads].to(kind)[:, None, None] * (key - place).abs()
                seen = key <= place
                if case["window"]:
                    seen &= key > place - case["window"]
                yield r, rows, heads, torch.where(seen, x, -math.inf)


def _prepare_sample(case, gen):
    rows, v = case["rows"], case["vocabulary"]
    x = torch.randn((rows, v), generator=gen, device=DEV) * case["spread"]
    x += 3 * torch.randn((rows, 1), generator=gen, device=DEV)
    few = torch.randint(0, v, (rows, 8), generator=gen, device=DEV)  # what the model is rather sure of
    x.scatter_add_(1, few, 2 * case["spread"] * torch.rand((rows, 8), generator=gen, device=DEV))
    state = {"case": case, "logits": x.to(DTYPES[case["dtype"]]),
             "uniforms": torch.rand((rows,), generator=gen, device=DEV)}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        state[name] = case[name]
        if case["mixed"]:  # a value for each request: some use the case's, some none; every fifth is greedy
            off = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}[name]
            on = torch.rand((rows,), generator=gen, device=DEV) < 0.7
            kind = torch.int32 if name == "top_k" else torch.float32
            state[name] = torch.where(on, case[name], off).to(kind)
            if name == "temperature":
                state[name][::5] = 0.0
    return state


# ------------------------------------------------------------------ the package's calls

def _own(s):
    case = s["case"]
    if case["op"] == "sample":
        from strict_topk_overlap_b200 import sampling
        return sampling.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                               top_p=s["top_p"], min_p=s["min_p"])
    from strict_topk_overlap_b200 import paged, paged_eviction
    cache = paged.PagedKVCache(s["k_pages"], s["v_pages"], s["table"], s["block_offsets"], s["lo"], s["hi"],
                               case["block"], case["page"], s["max_blocks"])
    if case["op"] == "weigh":
        return paged_eviction.accumulate_weights(s["weights"], s["q"], cache, s["lengths"], s["lse"],
                                                 token_offsets=s["token_offsets"], max_tokens=s["max_new"],
                                                 kv_lo=s["kv_lo"], softcap=case["cap"], slopes=s["slopes"])
    lengths, kept = paged_eviction.evict(cache, s["weights"], s["lengths"], case["keep"], first=case["first"],
                                         last=case["last"], weights_out=s["weights_out"])
    return {"lengths": lengths, "kept": kept, "weights": s["weights_out"], "k_pages": s["k_pages"],
            "v_pages": s["v_pages"], "lo": s["lo"], "hi": s["hi"]}


# ------------------------------------------------------------------ the plain forms

def _plain_weigh(s):
    case = s["case"]
    hkv, g, d, n, b = case["hkv"], case["hq"] // case["hkv"], case["d"], s["max_new"], case["block"]
    requests, ppb = case["requests"], b // case["page"]
    ends = None if s["token_offsets"] is None else s["token_offsets"].long()
    count = torch.ones((requests,), dtype=torch.long, device=DEV) if ends is None else ends.diff()
    start = torch.arange(requests, device=DEV) if ends is None else ends[:-1]
    i = torch.arange(n, device=DEV)
    token = torch.minimum(start[:, None] + i, (start + count - 1)[:, None])  # [R, n], the last one repeated
    at = (s["lengths"] - count)[:, None] + i
    room = s["block_offsets"].long().diff() * b
    slot = torch.arange(s["max_blocks"] * b, device=DEV)
    table = s["block_offsets"][:-1, None].long() * ppb + slot[::case["page"]] // case["page"]
    k = s["k_pages"][s["table"][table.clamp(max=s["table"].numel() - 1)].long()]  # [R, pages, Hkv, page, D]
    k = k.permute(0, 2, 1, 3, 4).flatten(2, 3).float()
    q = s["q"][token].float().view(requests, n, hkv, g, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (q @ k.transpose(-1, -2)).view(requests, hkv, g, n, -1) * d ** -0.5
    del k
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    place = at[:, None, None, :, None]
    if s["slopes"] is not None:
        x -= s["slopes"].view(hkv, g, 1, 1) * (place - slot).abs()
    x -= s["lse"][token].view(requests, n, hkv, g).permute(0, 2, 3, 1)[..., None]
    seen = (slot <= place) & (i < count[:, None])[:, None, None, :, None]
    if s["kv_lo"] is not None:
        seen &= slot >= s["kv_lo"][token][:, None, None, :, None]
    x = x.exp_().masked_fill_(~seen, 0.0).sum((2, 3))  # [R, Hkv, slots]
    to = torch.where(slot < room[:, None], s["block_offsets"][:-1, None] * b + slot, 0)
    x = x.masked_fill(~(slot < room[:, None])[:, None], 0.0)
    s["weights"].view(hkv, -1).scatter_add_(1, to.flatten().expand(hkv, -1), x.transpose(0, 1).flatten(1))
    return s["weights"]


def _plain_evict(s):
    case = s["case"]
    hkv, b, page, keep = case["hkv"], case["block"], case["page"], case["keep"]
    ppb, longest = b // page, s["max_blocks"] * b
    held, base = s["lengths"].long(), s["block_offsets"].long()
    slot = torch.arange(longest, device=DEV)
    there = (base[:-1, None] * b + slot).clamp(max=s["blocks"] * b - 1)  # [R, slots]
    w = s["weights"].view(hkv, -1)[:, there].transpose(0, 1)  # [R, Hkv, slots]
    end = held[:, None, None]
    w = torch.where((slot < case["first"]) | (slot >= end - case["last"]), math.inf, w)
    w = torch.where(slot < end, w, -1.0)  # (weights are not negative here)
    best = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :keep]
    if best.shape[-1] < keep:
        best = torch.cat((best, best.new_zeros((*best.shape[:2], keep - best.shape[-1]))), -1)
    best = best.sort(-1)[0]
    i = torch.arange(keep, device=DEV)
    kept = torch.where(end > keep, best, torch.where(i < end, i, -1))  # [R, Hkv, keep]
    lengths = held.clamp(max=keep)
    # Tokens kept[i] become tokens i. (Places without a token repeat token 0, which stays in a request that short.)
    source, goal = torch.where(kept < 0, 0, kept), torch.where(kept < 0, 0, i)
    head = torch.arange(hkv, device=DEV)[:, None]

    def where(x):
        return s["table"][base[:-1, None, None] * ppb + x // page].long(), head, x % page
    for pool in (s["k_pages"], s["v_pages"]):
        pool[where(goal)] = pool[where(source)]
    out = s["weights_out"].view(hkv, -1)
    moved = s["weights"].view(hkv, -1)[head, base[:-1, None, None] * b + source]
    out.zero_()
    out[head, base[:-1, None, None] * b + goal] = moved
    # Bounds of the requests that gave tokens up.
    block = torch.minimum(torch.arange(s["max_blocks"], device=DEV), base.diff()[:, None] - 1)  # [R, blocks], the last one repeated
    keys = s["k_pages"][s["table"][(base[:-1, None] + block)[..., None] * ppb + torch.arange(ppb, device=DEV)].long()].float()
    live = block[..., None] * b + torch.arange(b, device=DEV) < lengths[:, None, None]
    live, cut = live.view(*keys.shape[:3], 1, page, 1), (held > keep)[:, None, None]
    some = live.flatten(2).any(-1)[..., None, None]
    lo = torch.where(some, torch.where(live, keys, math.inf).amin((2, 4)), EMPTY)  # [R, blocks, Hkv, D]
    hi = torch.where(some, torch.where(live, keys, -math.inf).amax((2, 4)), -EMPTY)
    at = base[:-1, None] + block
    s["lo"][:, at] = torch.where(cut, lo.movedim(2, 0), s["lo"][:, at])
    s["hi"][:, at] = torch.where(cut, hi.movedim(2, 0), s["hi"][:, at])
    return {"lengths": lengths.int(), "kept": kept.int(), "weights": s["weights_out"], "k_pages": s["k_pages"],
            "v_pages": s["v_pages"], "lo": s["lo"], "hi": s["hi"]}


def _column(x, rows):
    """A parameter (FP32, or a whole number) as FP64 [rows, 1]."""
    x = x if isinstance(x, torch.Tensor) else torch.full((rows,), x, dtype=torch.float32, device=DEV)
    return x.double()[:, None]


def _plain_sample(s):
    x = s["logits"].double()
    rows, v = x.shape
    temperature, k, p, least = (_column(s[n], rows) for n in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = temperature == 0
    mass = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(v, device=DEV)
    mass = torch.where((rank < torch.where(greedy, 1.0, torch.where(k == 0, float(v), k))), mass, 0.0)
    before = mass.cumsum(-1) - mass
    mass = torch.where((before < p * mass.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0), mass, 0.0)
    mass = torch.where(mass >= least, mass, 0.0)
    mass = torch.zeros_like(mass).scatter_(1, order, mass).cumsum(-1)  # in the vocabulary's order
    passed = (mass <= s["uniforms"].double()[:, None] * mass[:, -1:]).sum(-1)
    return torch.minimum(passed, (mass < mass[:, -1:]).sum(-1)).int()


def run(state):
    if own:
        return _own(state)
    return {"weigh": _plain_weigh, "evict": _plain_evict, "sample": _plain_sample}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits

def _exact_sample(s):
    logits, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    rows, v = logits.shape
    get = {n: np.broadcast_to(s[n].cpu().numpy() if isinstance(s[n], torch.Tensor) else np.float32(s[n]), (rows,))
           for n in ("temperature", "top_k", "top_p", "min_p")}
    out = np.empty(rows, np.int32)
    for r in range(rows):
        x = logits[r]
        best = np.lexsort((np.arange(v), -x))
        if get["temperature"][r] == 0:
            out[r] = best[0]
            continue
        if get["top_k"][r]:
            best = best[:int(get["top_k"][r])]
        e = np.exp((x[best] - x[best[0]]) / np.float64(get["temperature"][r]))
        total = math.fsum(e)
        if get["top_p"][r] < 1:
            before = np.concatenate(([0.0], np.cumsum(e, dtype=np.longdouble)[:-1]))
            n = max(1, int((before < np.float64(get["top_p"][r]) * total).sum()))
            best, e = best[:n], e[:n]
        ok = e >= np.float64(get["min_p"][r])
        best, e = best[ok], e[ok]
        by = np.argsort(best)
        sums = np.cumsum(e[by], dtype=np.longdouble)
        out[r] = best[by][min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), len(by) - 1)]
    return torch.from_numpy(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    b, page, hkv = case["block"], case["page"], case["hkv"]
    ppb, offsets = b // page, s["block_offsets"].tolist()
    weights = s["weights"].double().view(hkv, -1)
    if case["op"] == "weigh":
        g = case["hq"] // hkv
        for r, rows, heads, x in _parts(s, *_lengths(case), torch.float64):
            share = torch.exp(x - s["lse"][rows, heads].double().t()[..., None]).sum((0, 1))
            weights[heads.start // g, offsets[r] * b:offsets[r] * b + share.numel()] += share
        return weights.view(s["weights"].shape)
    out = {n: s[n].double() for n in ("k_pages", "v_pages", "lo", "hi")}
    keep, first, last = case["keep"], case["first"], case["last"]
    every = torch.full((case["requests"], hkv, keep), -1, dtype=torch.int32, device=DEV)
    fresh = torch.zeros_like(weights)
    for r, n in enumerate(_held(case)):
        pages = s["table"].long()[offsets[r] * ppb:offsets[r + 1] * ppb]
        for h in range(hkv):
            row = weights[h, offsets[r] * b:offsets[r] * b + n]
            kept = torch.arange(n, device=DEV)
            if n > keep:
                middle = torch.argsort(row[first:n - last], descending=True, stable=True)[:keep - first - last] + first
                kept = torch.cat((kept[:first], middle, kept[n - last:])).sort()[0]
            every[r, h, :kept.numel()] = kept
            fresh[h, offsets[r] * b:offsets[r] * b + kept.numel()] = row[kept]
            if n <= keep:
                continue
            to = torch.arange(keep, device=DEV)
            for name in ("k_pages", "v_pages"):
                pool = out[name]
                pool[pages[to // page], h, to % page] = pool[pages[kept // page], h, kept % page].clone()
            keys = out["k_pages"][pages, h].reshape(-1, case["d"])
            blocks = offsets[r + 1] - offsets[r]
            full = -(-keep // b)
            for name, fill, pick in (("lo", EMPTY, torch.amin), ("hi", -EMPTY, torch.amax)):
                edge = math.inf if name == "lo" else -math.inf
                x = torch.where((torch.arange(full * b, device=DEV) < keep)[:, None], keys[:full * b], edge)
                out[name][h, offsets[r]:offsets[r] + full] = pick(x.view(full, b, -1), 1)
                out[name][h, offsets[r] + full:offsets[r] + blocks] = float(np.float32(fill))
    lengths = torch.tensor([min(n, keep) for n in _held(case)], dtype=torch.int32, device=DEV)
    return {"lengths": lengths, "kept": every, "weights": fresh.view(s["weights"].shape), **out}
