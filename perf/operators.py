"""Cases for the dense side of a paged decode service: appending rotated keys
and values to the page pool, attention of prompts and of single tokens over
it, and attention of a batch whose requests share a long prefix.

``run`` computes each operator in elementary torch operations in FP32 (rounded
once at the end), or, with ``own`` set, through the package's entry points on
the same inputs. Page pools are [pages, Hkv, page, D], block g of the batch is
made of the pages page_table[g * block / page + i], and request r owns the
blocks block_offsets[r] .. block_offsets[r + 1]. New tokens are packed
request after request (request r: token_offsets[r] .. token_offsets[r + 1]).
"""
from __future__ import annotations

import bisect
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def _case(name, op, dtype, hq, hkv, d, block, page, requests, past, new, **more):
    case = {"op": op, "dtype": dtype, "hq": hq, "hkv": hkv, "d": d, "block": block, "page": page,
            "requests": requests, "past_min": past[0], "past_max": past[1], "new_min": new[0], "new_max": new[1],
            "shape_seed": 7, **more}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One decode step of a small batch: eight tokens rotated and appended. Latency is what counts.
        _case("append-step-8", "append", "bf16", 32, 8, 128, 32, 16, 8, (1000, 5000), (1, 1),
              rotary=128, interleaved=False, axes=1),
        # Five prompts of odd lengths enter the cache, one of them behind tokens that are there already.
        _case("append-prompts", "append", "bf16", 32, 8, 128, 32, 16, 5, (0, 700), (1, 4097),
              rotary=128, interleaved=False, axes=1),
        # Two long video prompts: (time, height, width) positions.
        _case("append-video", "append", "f16", 16, 8, 128, 32, 16, 2, (0, 0), (15000, 17000),
              rotary=128, interleaved=False, axes=3),
        # Three prompts with capped scores, causal.
        _case("prompt-capped", "attend", "bf16", 16, 8, 128, 32, 16, 3, (0, 0), (1500, 8192), mask="causal", cap=50.0,
              slopes=False),
        # The last piece of a long prompt, its scores biased by distance.
        _case("prompt-piece-biased", "attend", "bf16", 32, 8, 128, 32, 16, 1, (65000, 65000), (509, 509),
              mask="causal", cap=0.0, slopes=True),
        # Documents packed into one sequence, each blind to the others.
        _case("prompt-documents", "attend", "f16", 32, 8, 64, 32, 16, 1, (0, 0), (8191, 8191), mask="documents",
              cap=0.0, slopes=False),
        # Prompts whose first part sees all of itself (an image, an instruction), wide head groups.
        _case("prompt-prefix", "attend", "bf16", 96, 8, 128, 32, 32, 3, (0, 0), (200, 2300), mask="prefix", cap=0.0,
              slopes=False),
        # One token for each of 64 requests of 8 K to 32 K tokens.
        _case("token-batch-64", "attend", "bf16", 16, 8, 128, 32, 16, 64, (8191, 32767), (1, 1), mask="causal",
              cap=0.0, slopes=False),
        # One token of one long request, capped: the split over the context is what counts.
        _case("token-one-long", "attend", "bf16", 32, 8, 128, 32, 16, 1, (65535, 65535), (1, 1), mask="causal",
              cap=50.0, slopes=False),
        # The smallest decode call, in FP32.
        _case("token-one-f32", "attend", "f32", 8, 2, 128, 32, 16, 1, (4095, 4095), (1, 1), mask="causal", cap=0.0,
              slopes=False),
        # 64 requests behind one system prompt of 32 K tokens.
        _case("shared-64", "shared", "bf16", 32, 8, 128, 32, 16, 64, (0, 1023), (1, 1), prefix=32768, cap=0.0,
              slopes=False),
        # A few requests of a small model behind a short shared prefix, three tokens each (drafts to be verified).
        _case("shared-7-drafts", "shared", "f16", 8, 2, 128, 32, 16, 7, (0, 500), (3, 3), prefix=4096, cap=0.0,
              slopes=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "prompt", "token", "shared"))
    hq, hkv = rng.choice(((32, 8), (16, 8), (8, 2), (96, 8), (8, 8)))
    d = rng.choice((64, 128))
    page = rng.choice((16, 32))
    block = rng.choice((32, 64))
    kind = rng.choice(("bf16", "f16"))
    seed = rng.randrange(1 << 20)
    while True:
        if op == "append":
            requests = _log(rng, 1, 64)
            top = _log(rng, 1, 30000)
            past = _log(rng, 1, 8000)
            case = _case(None, "append", rng.choice(("bf16", "f16", "f32")), hq, hkv, d, block, page, requests,
                         (0, past), (1, top), rotary=rng.choice((d, d, d // 2)), interleaved=rng.random() < 0.5,
                         axes=rng.choice((1, 3)), shape_seed=seed)
            if sum(_lengths(case)[1]) * (hq + 2 * hkv) * d <= 33000 * 32 * 128:
                return case
        elif op == "prompt":
            requests = _log(rng, 1, 8)
            top = _log(rng, 32, 8000)
            past = rng.choice((0, 0, _log(rng, 32, 32000)))
            case = _case(None, "attend", kind, hq, hkv, d, block, page, requests, (past // 2, past), (1, top),
                         mask=rng.choice(("causal", "documents", "prefix", "window")),
                         cap=rng.choice((0.0, 30.0, 50.0)), slopes=rng.random() < 0.3, shape_seed=seed)
            if requests * hq * top * (top + past) * d <= 3 * 16 * 8192 * 8192 * 128:
                return case
        elif op == "token":
            requests = _log(rng, 1, 64)
            top = _log(rng, 64, 65536)
            case = _case(None, "attend", rng.choice(("bf16", "f16", "f32")), hq, hkv, d, block, page, requests,
                         (top // 4, top), (1, 1), mask=rng.choice(("causal", "causal", "window")),
                         cap=rng.choice((0.0, 50.0)), slopes=rng.random() < 0.3, shape_seed=seed)
            if requests * top * hkv * d * (2 if case["dtype"] == "f32" else 1) <= 64 * 20000 * 8 * 128:
                return case
        else:
            requests = _log(rng, 2, 64)
            prefix = block * (2 * _log(rng, 8, 500) + 1)
            case = _case(None, "shared", kind, hq, hkv, d, block, page, requests, (0, _log(rng, 1, 1024)),
                         rng.choice(((1, 1), (1, 1), (4, 4))), prefix=prefix, cap=rng.choice((0.0, 50.0)),
                         slopes=rng.random() < 0.2, shape_seed=seed)
            if requests * case["new_max"] * hq * prefix * d <= 64 * 32 * 32768 * 128:
                return case


def _lengths(case):
    """Tokens in the cache before the call, and new ones, per request."""
    rng = random.Random(case["shape_seed"])
    past = [rng.randint(case["past_min"], case["past_max"]) for _ in range(case["requests"])]
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["requests"])]
    return [p + case.get("prefix", 0) for p in past], new


def _intervals(case):
    """[lo, hi) of the keys that each new token sees, as two lists over the packed tokens."""
    rng = random.Random(case["shape_seed"] + 1)
    lo, hi = [], []
    for p, n in zip(*_lengths(case)):
        at = range(p, p + n)
        mask = case.get("mask", "causal")
        if mask == "documents":
            starts = [0]
            while starts[-1] < p + n:
                starts.append(starts[-1] + rng.randint(1, max(2, (p + n) // 4)))
            lo += [starts[bisect.bisect_right(starts, i) - 1] for i in at]
            hi += [i + 1 for i in at]
        elif mask == "prefix":
            whole = rng.randint(1, p + n)
            lo += [0] * n
            hi += [max(i + 1, whole) for i in at]
        elif mask == "window":
            width = rng.randint(1, max(2, (p + n) // 2))
            lo += [max(0, i + 1 - width) for i in at]
            hi += [i + 1 for i in at]
        else:
            lo += [0] * n
            hi += [i + 1 for i in at]
    return lo, hi


def _cumulative(counts):
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return total


def work(case):
    past, new = _lengths(case)
    t, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["d"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        b = case["block"]
        touched = sum((p + n - 1) // b - p // b + 1 for p, n in zip(past, new))
        moved = 2 * t * (hq + 2 * hkv) * d * size + 2 * touched * hkv * d * 4 + t * case["rotary"] * 4
        return {"bytes": moved + t * case["axes"] * 4, "flops": 3 * t * (hq + hkv) * case["rotary"]}
    lo, hi = _intervals(case)
    pairs = sum(max(0, y - x) for x, y in zip(lo, hi))
    at = _cumulative(new)
    seen = sum(max(hi[a:z]) - min(lo[a:z]) for a, z in zip(at, at[1:]))
    seen -= (case["requests"] - 1) * case.get("prefix", 0)
    return {"bytes": 2 * t * hq * d * size + 2 * seen * hkv * d * size, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _pool(case, gen, pages):
    """Keys N(0, 1) with a bias per page, N(0, 0.5^2) (neighbouring tokens are alike), and values N(0, 1)."""
    shape = (pages, case["hkv"], case["page"], case["d"])
    dtype = DTYPES[case["dtype"]]
    k = torch.randn(shape, generator=gen, device=DEV, dtype=dtype)
    k += 0.5 * torch.randn((pages, case["hkv"], 1, case["d"]), generator=gen, device=DEV, dtype=dtype)
    return k, torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    past, new = _lengths(case)
    b, ppb, hkv, hq, d = case["block"], case["block"] // case["page"], case["hkv"], case["hq"], case["d"]
    dtype, t = DTYPES[case["dtype"]], sum(new)
    blocks = [-(-(p + n) // b) for p, n in zip(past, new)]
    shared = case.get("prefix", 0) // b  # blocks that every request's table begins with
    offsets = _cumulative(blocks)
    pages = (shared + sum(n - shared for n in blocks)) * ppb
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)  # as an allocator leaves them
    if shared:
        rows, at = [], shared
        for n in blocks:
            rows += [order[:shared * ppb], order[at * ppb:(at + n - shared) * ppb]]
            at += n - shared
        table = torch.cat(rows)
    else:
        table = order
    k_pages, v_pages = _pool(case, gen, pages)
    state = {"case": case, "k_pages": k_pages, "v_pages": v_pages, "table": table,
             "block_offsets": _ints(offsets), "max_blocks": max(blocks), "max_new": max(new),
             "token_offsets": None if max(new) == 1 else _ints(_cumulative(new))}
    if case["op"] == "append":
        qkv = torch.randn((t, hq + 2 * hkv, d), generator=gen, device=DEV, dtype=dtype)  # one projection's output
        state |= {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:], "lengths": _ints(past)}
        # Bounds of the cached tokens of each block (a block without any keeps whatever it has).
        cached = k_pages[table.long()].view(-1, ppb, hkv, case["page"], d)
        filled = torch.cat([(torch.arange(n * b) < p) for n, p in zip(blocks, past)]).to(DEV)
        filled = filled.view(-1, ppb, 1, case["page"], 1)
        state["lo"] = cached.float().masked_fill(~filled, 3e38).amin((1, 3)).transpose(0, 1).contiguous()
        state["hi"] = cached.float().masked_fill(~filled, -3e38).amax((1, 3)).transpose(0, 1).contiguous()
        half = case["rotary"] // 2
        rate = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(max(p + n for p, n in zip(past, new)), dtype=torch.float64)[:, None] * rate
        state["cos"], state["sin"] = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
        state["positions"] = state["axis"] = None
        if case["axes"] == 3:  # frames of 24 x 32 patches
            at = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)])
            state["positions"] = torch.stack([at // 768, at // 32 % 24, at % 32]).to(torch.int32).to(DEV)
            state["axis"] = torch.tensor([0 if i < half // 4 else 1 if i < half * 5 // 8 else 2 for i in range(half)],
                                         dtype=torch.uint8).to(DEV)
        return state
    none = torch.empty((hkv, 0, d), device=DEV)  # a cache that no block selection reads keeps no bounds
    state |= {"lo": none, "hi": none, "lengths": _ints([p + n for p, n in zip(past, new)])}
    state["q"] = torch.randn((t, hq, d), generator=gen, device=DEV, dtype=dtype)
    state["kv_lo"] = state["kv_hi"] = state["slopes"] = None
    lo, hi = _intervals(case)
    if case.get("mask") in ("documents", "window"):
        state["kv_lo"] = _ints(lo)
    if case.get("mask") == "prefix":
        state["kv_hi"] = _ints(hi)
    if case["slopes"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV)
    return state


# ------------------------------------------------------------------ the package's calls

def _own(s):
    from strict_topk_overlap_b200 import paged, paged_append, paged_attention, rotary
    case = s["case"]
    cache = paged.PagedKVCache(s["k_pages"], s["v_pages"], s["table"], s["block_offsets"], s["lo"], s["hi"],
                               case["block"], case["page"], s["max_blocks"])
    if case["op"] == "append":
        turn = rotary.Rotary(s["cos"], s["sin"], interleaved=case["interleaved"], axis=s["axis"])
        q = paged_append.append_tokens(cache, s["k"], s["v"], s["lengths"], token_offsets=s["token_offsets"],
                                       q=s["q"], rotary=turn, positions=s["positions"])
        return {"q": q, "k_pages": cache.k_pages, "v_pages": cache.v_pages, "lo": cache.lo, "hi": cache.hi}
    more = {"token_offsets": s["token_offsets"], "max_tokens": s["max_new"], "softcap": case["cap"],
            "slopes": s["slopes"]}
    if case["op"] == "shared":
        return paged_attention.shared_prefix_attention(s["q"], cache, s["lengths"], case["prefix"], **more)
    return paged_attention.attention(s["q"], cache, s["lengths"], kv_lo=s["kv_lo"], kv_hi=s["kv_hi"], **more)


# ------------------------------------------------------------------ the plain forms

def _requests_of(s, t):
    """Request and place among its new tokens, of each packed token."""
    at = torch.arange(t, device=DEV)
    if s["token_offsets"] is None:
        return at, torch.zeros_like(at)
    r = torch.searchsorted(s["token_offsets"][1:].long(), at, right=True)
    return r, at - s["token_offsets"][r]


def _turned(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] dims of x [T, H, D] rotated pair by pair, in FP32."""
    half = cos.shape[-1]
    x = x.float()
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, z = head[..., 0::2], head[..., 1::2]
    else:
        a, z = head[..., :half], head[..., half:]
    c, n = cos[:, None], sin[:, None]
    one, two = a * c - z * n, z * c + a * n
    head = torch.stack((one, two), -1).flatten(-2) if interleaved else torch.cat((one, two), -1)
    return torch.cat((head, rest), -1)


def _plain_append(s):
    case, t, dtype = s["case"], s["k"].shape[0], s["k"].dtype
    b, page, ppb = case["block"], case["page"], case["block"] // case["page"]
    r, i = _requests_of(s, t)
    at = s["lengths"][r].long() + i
    if s["positions"] is None:
        cos, sin = s["cos"][at], s["sin"][at]
    else:
        pair = torch.arange(s["cos"].shape[1], device=DEV)
        own_position = s["positions"][s["axis"].long()].t().long()  # [T, pairs]
        cos, sin = s["cos"][own_position, pair], s["sin"][own_position, pair]
    q = _turned(s["q"], cos, sin, case["interleaved"]).to(dtype)
    k = _turned(s["k"], cos, sin, case["interleaved"]).to(dtype)
    block = s["block_offsets"][r] + at // b
    where = s["table"][block * ppb + at % b // page].long()
    s["k_pages"][where, :, at % page] = k
    s["v_pages"][where, :, at % page] = s["v"]
    # Bounds of the blocks that got tokens, over all their tokens.
    new = s["lengths"] * 0 + 1 if s["token_offsets"] is None else s["token_offsets"].diff()
    end = (s["lengths"] + new)[:, None].long()
    touched = s["lengths"][:, None].long() // b + torch.arange((s["max_new"] + b - 2) // b + 1, device=DEV)
    touched = torch.minimum(touched, (end - 1) // b)
    block = s["block_offsets"][:-1, None] + touched
    where = s["table"][block[..., None] * ppb + torch.arange(ppb, device=DEV)].long()
    keys = s["k_pages"][where].float()  # [R, blocks, ppb, Hkv, page, D]
    place = touched[..., None] * b + torch.arange(b, device=DEV)
    live = (place < end[..., None]).view(*where.shape, 1, page, 1)
    inf = float("inf")
    s["lo"][:, block] = torch.where(live, keys, inf).amin((2, 4)).movedim(2, 0)
    s["hi"][:, block] = torch.where(live, keys, -inf).amax((2, 4)).movedim(2, 0)
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "lo": s["lo"], "hi": s["hi"]}


def _tokens(s, pages, first, count):
    """Tokens [first, first + count) of every request (whole pages), FP32 [R, Hkv, count, D]."""
    case = s["case"]
    page, ppb = case["page"], case["block"] // case["page"]
    at = s["block_offsets"][:-1, None].long() * ppb + torch.arange(first // page, (first + count) // page, device=DEV)
    got = pages[s["table"][at.clamp(max=s["table"].numel() - 1)].long()]  # [R, pages, Hkv, page, D]
    return got.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _scores(s, x, place, row_place, seen_lo, seen_hi):
    """Scaled, capped, biased and masked scores. x [.., G, n, keys] with the KV heads before G."""
    case = s["case"]
    x = x * case["d"] ** -0.5
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    if s["slopes"] is not None:
        steep = s["slopes"].view(case["hkv"], -1, 1, 1)
        x = x - steep * (row_place[..., None] - place).abs()
    return x.masked_fill((place < seen_lo[..., None]) | (place >= seen_hi[..., None]), float("-inf"))


def _plain_attend(s):
    case, t = s["case"], s["q"].shape[0]
    hkv, g, d, n = case["hkv"], case["hq"] // case["hkv"], case["d"], s["max_new"]
    r, i = _requests_of(s, t)
    count = s["lengths"] * 0 + 1 if s["token_offsets"] is None else s["token_offsets"].diff()
    start = torch.arange(case["requests"], device=DEV) if s["token_offsets"] is None else s["token_offsets"][:-1]
    token = torch.minimum(start[:, None] + torch.arange(n, device=DEV), (start + count - 1)[:, None]).long()  # [R, n]
    q = s["q"][token].float().view(-1, n, hkv, g, d).permute(0, 2, 3, 1, 4)  # [R, Hkv, G, n, D]
    at = (s["lengths"] - count)[:, None] + torch.arange(n, device=DEV)
    seen_lo = torch.zeros_like(at) if s.get("kv_lo") is None else s["kv_lo"][token]
    seen_hi = at + 1 if s.get("kv_hi") is None else s["kv_hi"][token]
    row = lambda x: x[:, None, None]  # noqa: E731
    length = s["max_blocks"] * case["block"]
    prefix = case.get("prefix", 0)
    place = torch.arange(length, device=DEV)
    k = _tokens(s, s["k_pages"], prefix, length - prefix)
    x = (q.flatten(2, 3) @ k.transpose(-1, -2)).view(*q.shape[:4], -1)
    x = _scores(s, x, place[prefix:], row(at), row(seen_lo), row(seen_hi))
    del k
    if prefix:  # the same keys for all: one product of all the queries
        first = {**s, "block_offsets": s["block_offsets"][:2]}
        every = q.permute(1, 0, 2, 3, 4)
        y = every.flatten(1, 3) @ _tokens(first, s["k_pages"], 0, prefix)[0].transpose(-1, -2)
        y = y.view(*every.shape[:4], -1).permute(1, 0, 2, 3, 4)
        x = torch.cat((_scores(s, y, place[:prefix], row(at), row(seen_lo), row(seen_hi)), x), -1)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    total = x.sum(-1, keepdim=True)
    out = (x[..., prefix:].flatten(2, 3) @ _tokens(s, s["v_pages"], prefix, length - prefix)).view(q.shape)
    if prefix:
        every = x[..., :prefix].permute(1, 0, 2, 3, 4)
        y = every.flatten(1, 3) @ _tokens(first, s["v_pages"], 0, prefix)[0]
        out = out + y.view(*every.shape[:4], d).permute(1, 0, 2, 3, 4)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[r, i].to(s["q"].dtype)


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attend(state)


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lengths(case)
    b, page, hkv, d = case["block"], case["page"], case["hkv"], case["d"]
    ppb, g = b // page, case["hq"] // case["hkv"]
    offsets, start = s["block_offsets"].tolist(), _cumulative(new)
    if case["op"] == "append":
        out = {n: s[n].double() for n in ("q", "k_pages", "v_pages", "lo", "hi")}
        for r, (p, n) in enumerate(zip(past, new)):
            for at in range(0, n, 4096):
                m = min(4096, n - at)
                rows = slice(start[r] + at, start[r] + at + m)
                place = torch.arange(p + at, p + at + m, device=DEV)
                half = case["rotary"] // 2
                if s["positions"] is None:
                    index = place[:, None].expand(m, half)
                else:
                    index = torch.stack([s["positions"][int(a), rows] for a in s["axis"].tolist()], 1).long()
                c = s["cos"].double().gather(0, index)[:, None]
                w = s["sin"].double().gather(0, index)[:, None]
                first = torch.arange(half, device=DEV) * (2 if case["interleaved"] else 1)
                second = first + (1 if case["interleaved"] else half)
                turned = {}
                for name in ("q", "k"):
                    x = s[name][rows].double()
                    y = x.clone()
                    y[..., first] = x[..., first] * c - x[..., second] * w
                    y[..., second] = x[..., first] * w + x[..., second] * c
                    turned[name] = y
                out["q"][rows] = turned["q"]
                pages = s["table"].long()[offsets[r] * ppb + place // page]
                out["k_pages"][pages, :, place % page] = turned["k"]
                out["v_pages"][pages, :, place % page] = s["v"][rows].double()
            for j in range(p // b, (p + n - 1) // b + 1):  # the bounds are those of the keys as they are stored
                pages = s["table"].long()[(offsets[r] + j) * ppb:(offsets[r] + j + 1) * ppb]
                keys = out["k_pages"][pages].transpose(1, 2).reshape(b, hkv, d)[:p + n - j * b]
                keys = keys.to(s["k"].dtype).double()
                out["lo"][:, offsets[r] + j], out["hi"][:, offsets[r] + j] = keys.amin(0), keys.amax(0)
        return out
    lo, hi = (torch.tensor(x, device=DEV) for x in _intervals(case))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, (p, n) in enumerate(zip(past, new)):
        pages = s["table"].long()[offsets[r] * ppb:offsets[r + 1] * ppb]
        for h in range(hkv):
            k = s["k_pages"][pages, h].reshape(-1, d)[:p + n].double()
            v = s["v_pages"][pages, h].reshape(-1, d)[:p + n].double()
            for at in range(0, n, 2048):
                rows = torch.arange(start[r] + at, start[r] + min(n, at + 2048), device=DEV)
                place = p + rows - start[r]
                x = s["q"][rows, h * g:(h + 1) * g].double().transpose(0, 1) @ k.t() / math.sqrt(d)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                key = torch.arange(p + n, device=DEV)
                if s["slopes"] is not None:
                    x -= s["slopes"][h * g:(h + 1) * g].double()[:, None, None] * (key - place[:, None]).abs()
                seen = (key >= lo[rows][:, None]) & (key < hi[rows][:, None])
                x = torch.where(seen, x, float("-inf"))
                share = torch.softmax(x, -1).nan_to_num(0.0)
                out[rows, h * g:(h + 1) * g] = (share @ v).transpose(0, 1)
    return out
