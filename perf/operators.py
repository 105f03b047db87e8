"""Serving from a paged cache that holds keys and values in 8 bits: the operators, their plain forms and the work they are asked for.

Four paths: `tables` (page tables, slots and positions of a ragged batch, from request lengths), `rotary` (rotary positions of
queries and keys, and their gradient), `append` (new keys and values into the cache) and `attention` (over the cache: single
tokens, chunks of prompts, an encoder's states).  The cache: e4m3 values k (pages, kv_heads, page_size, head_dim) and
v (pages, kv_heads, head_dim, page_size), with one power of two per page and head each.  Slot = page * page_size + place in it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

E4M3 = torch.float8_e4m3fn
LARGEST, SMALLEST_SCALE = 448.0, 2.0 ** -118  # of an e4m3 value; of a page whose values are all zero


def listed():
    return [
        # A decode step's bookkeeping: 64 requests of all ages, one new token each.
        {"name": "tables_decode_64", "path": "tables", "requests": 64, "page": 64, "longest": 4096, "prompts": 0, "fresh": 1},
        # A large mixed step on small pages: 1024 requests, 64 of them with prompts of up to 512 tokens.
        {"name": "tables_mixed_1024", "path": "tables", "requests": 1024, "page": 16, "longest": 8192, "prompts": 64, "fresh": 512},
        # Queries and keys of a decode step, in place in the fused projection of 32 + 2 x 8 heads, far positions, scaled for them.
        {"name": "rotary_16_rows", "path": "rotary", "rows": 16, "heads": 40, "row_heads": 48, "dim": 128, "rotary": 128,
         "interleaved": False, "type": "bf16", "farthest": 131072, "factor": 8.0, "by_parts": True, "gradient": False},
        # The same for the prompts of a step.
        {"name": "rotary_8192_rows", "path": "rotary", "rows": 8192, "heads": 40, "row_heads": 48, "dim": 128, "rotary": 128,
         "interleaved": False, "type": "bf16", "farthest": 32768, "factor": 1.0, "by_parts": False, "gradient": False},
        # Training in f32 on the decoder's batch (16 x 1024 tokens, queries and keys of 8 heads of 64): forward and gradient,
        # half of each head turned, neighbours paired.
        {"name": "rotary_train_16384", "path": "rotary", "rows": 16384, "heads": 16, "row_heads": 24, "dim": 64, "rotary": 32,
         "interleaved": True, "type": "f32", "farthest": 1024, "factor": 1.0, "by_parts": False, "gradient": True},
        # A decode step's keys and values in f32: one row each of 77 requests, into small pages that are partly full.
        {"name": "append_77_rows_f32", "path": "append", "requests": 77, "fresh": 1, "cached": 500, "page": 16, "kv_heads": 5, "dim": 64,
         "type": "f32"},
        # Prompts: 8192 rows of 16 requests.
        {"name": "append_8192_rows", "path": "append", "requests": 16, "fresh": 512, "cached": 200, "page": 64, "kv_heads": 8, "dim": 128,
         "type": "bf16"},
        # One user's next token.
        {"name": "decode_1x4097", "path": "attention", "requests": 1, "shortest": 4097, "longest": 4097, "fresh": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True},
        # The next tokens of 64 users with contexts of all lengths.
        {"name": "decode_64x8192", "path": "attention", "requests": 64, "shortest": 16, "longest": 8192, "fresh": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True},
        # The next tokens of two users with a long document each: few rows, keys without end.
        {"name": "decode_2x131072", "path": "attention", "requests": 2, "shortest": 131072, "longest": 131072, "fresh": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True},
        # Chunks of prompts behind what is cached of them: 8 requests, 500 tokens each.
        {"name": "prefill_8x500", "path": "attention", "requests": 8, "shortest": 1000, "longest": 4000, "fresh": 500, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True},
        # A decoder's tokens over an encoder's cached states, a head of keys for each of queries.
        {"name": "cross_16x1500", "path": "attention", "requests": 16, "shortest": 1500, "longest": 1500, "fresh": 1, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 32, "causal": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


# No drawn case asks for more than its path's largest listed one does.
_MOST_BYTES = {"tables": 4e5, "rotary": 4.1e8, "append": 6e7, "attention": 5.6e8}
_MOST_FLOPS = 1.3e11


def draw(rng):
    path = rng.choice(["tables", "rotary", "append", "attention", "attention"])
    while True:
        case = {"path": path}
        if path == "tables":
            requests = _log(rng, 1, 1024)
            case.update(requests=requests, page=rng.choice([16, 32, 64, 128, 256]), longest=_log(rng, 16, 8192),
                        prompts=rng.choice([0, requests // 16, requests]), fresh=_log(rng, 1, 512))
        elif path == "rotary":
            dim = rng.choice([64, 80, 96, 128, 256])
            heads = _log(rng, 1, 48)
            case.update(rows=_log(rng, 1, 16384), heads=heads, row_heads=heads + rng.choice([0, 1, heads]), dim=dim,
                        rotary=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                        type=rng.choice(["bf16", "bf16", "f32"]), farthest=_log(rng, 16, 131072), factor=rng.choice([1.0, 4.0, 8.0]),
                        by_parts=rng.random() < 0.5, gradient=rng.random() < 0.4)
        elif path == "append":
            case.update(requests=_log(rng, 1, 128), fresh=_log(rng, 1, 1024), cached=_log(rng, 1, 1000),
                        page=rng.choice([16, 32, 64, 128, 256]), kv_heads=_log(rng, 1, 16), dim=rng.choice([64, 128, 256]),
                        type=rng.choice(["bf16", "bf16", "f32"]))
        else:
            kv_heads, longest = _log(rng, 1, 16), _log(rng, 16, 16384)
            case.update(requests=_log(rng, 1, 64), shortest=_log(rng, 1, longest), longest=longest,
                        fresh=rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 700)]), heads=kv_heads * rng.choice([1, 2, 4, 5, 8, 16]),
                        kv_heads=kv_heads, dim=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128, 256]),
                        causal=rng.random() < 0.8)
        if _affordable(case):
            return case


def _affordable(case):
    cost = work(case)
    if case["path"] == "attention":  # the plain form holds all the scores, and every request's keys at the longest one's length
        padded = case["requests"] * (case["longest"] + case["fresh"] + 256)
        if padded * case["kv_heads"] * case["dim"] > 7e8 or padded * case["heads"] * case["fresh"] > 7e8:
            return False
    if case["path"] == "append" and case["requests"] * (case["fresh"] + case["cached"]) * case["kv_heads"] * case["dim"] > 1e8:
        return False
    return cost["bytes"] <= _MOST_BYTES[case["path"]] and cost["flops"] <= _MOST_FLOPS


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _spread(low, high, count):
    """`count` lengths of low..high, evenly spaced in their logarithm."""
    at = (np.arange(count) + 0.5) / count
    return np.clip(np.exp(math.log(low) + at * math.log((high + 1) / low)).astype(np.int64), low, high)


def _lengths(case, seed):
    """What each request has in the cache and how many new rows it brings, as host arrays: lengths of the case, in an order of the seed."""
    rng, n = np.random.default_rng(seed), case["requests"]
    if case["path"] == "tables":
        cached, fresh = rng.permutation(_spread(1, case["longest"], n)), np.ones(n, np.int64)
        if case["prompts"]:
            with_prompt = rng.permutation(n)[:case["prompts"]]
            fresh[with_prompt] = np.linspace(1, case["fresh"], len(with_prompt)).astype(np.int64)
            cached[with_prompt[::2]] = 0  # half of them begin here
        return cached, fresh
    fresh = np.full(n, case["fresh"], np.int64)
    if case["path"] == "append":
        return rng.permutation(np.linspace(case["cached"] // 2, case["cached"], n).astype(np.int64)), fresh
    after = rng.permutation(_spread(case["shortest"], case["longest"], n))
    return np.maximum(after - fresh, 0) if case["causal"] else after, fresh


def _pages(count, page):
    return (count + page - 1) // page


def _table(rng, used, spare, width):
    """A page table with the given number of pages for each request, scattered over a cache of `spare` pages more; -1 behind them."""
    pages = int(used.sum()) + spare
    order, table, at = rng.permutation(pages), np.full((len(used), width), -1, np.int64), 0
    for r, count in enumerate(used):
        table[r, :count] = order[at:at + count]
        at += count
    return pages, table


def _codes(generator, *shape):
    """e4m3 values as a page holds them: the largest of some thousand normal values near the end of the range."""
    x = torch.randn(*shape, generator=generator, device="cuda").mul_(100.0).clamp_(-LARGEST, LARGEST)
    return x.to(E4M3)


def _scales(generator, *shape):
    return torch.exp2(torch.randint(-8, -5, shape, generator=generator, device="cuda").float())


def prepare(case, seed):
    path, s = case["path"], {"case": case}
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    kind = torch.float32 if case.get("type") == "f32" else torch.bfloat16
    if path == "rotary":
        rows, width = case["rows"], case["row_heads"] * case["dim"]
        make = lambda: torch.randn(rows, width, generator=generator, device="cuda").to(kind)
        s.update(x=make(), positions=torch.randint(0, case["farthest"], (rows,), generator=generator, device="cuda").int(),
                 out=torch.empty(rows, case["heads"], case["dim"], device="cuda", dtype=kind))
        if case["gradient"]:
            s.update(g=torch.randn(rows, case["heads"], case["dim"], generator=generator, device="cuda").to(kind),
                     gx=torch.empty(rows, case["heads"], case["dim"], device="cuda", dtype=kind))
        return s
    cached, fresh = _lengths(case, seed)
    page, rng = case["page"], np.random.default_rng(seed + 1)
    if path == "tables":
        had, used = _pages(cached, page), _pages(cached + fresh, page)
        pages, table = _table(rng, used, 0, _pages(case["longest"] + case["fresh"], page))
        dealt = rng.permutation(np.concatenate([table[r, had[r]:used[r]] for r in range(len(used))])) if (used > had).any() else np.zeros(0, np.int64)
        free = np.concatenate([dealt, pages + rng.permutation(32)])
        table[np.arange(table.shape[1])[None] >= had[:, None]] = -1
        rows = int(fresh.sum())
        new = lambda n: torch.full((n,), -1, dtype=torch.int32, device="cuda")
        s.update(cached=_ints(cached), fresh=_ints(fresh), free=_ints(free), table=_ints(table), rows=rows, row_offsets=new(len(used) + 1),
                 lengths=new(len(used)), positions=new(rows), slots=new(rows), counts=new(3))
        return s
    after = cached + fresh if path == "append" or case["causal"] else cached
    used = _pages(after, page)
    pages, table = _table(rng, used, 3, max(1, int(used.max())))
    heads, dim = case["kv_heads"], case["dim"]
    s.update(pages=pages, k=_codes(generator, pages, heads, page, dim), v=_codes(generator, pages, heads, dim, page),
             k_scales=_scales(generator, pages, heads), v_scales=_scales(generator, pages, heads))
    rows = int(fresh.sum())
    if path == "append":
        request = np.repeat(np.arange(len(fresh)), fresh)
        place = cached[request] + np.arange(rows) - (np.cumsum(fresh) - fresh)[request]
        # Rows of the fused projection of as many query heads: keys and values stand behind them.  Their sizes differ from row to row.
        qkv = torch.randn(rows, 3 * heads * dim, generator=generator, device="cuda")
        qkv *= torch.exp2(torch.randint(-1, 2, (rows, 1), generator=generator, device="cuda").float())
        s.update(qkv=qkv.to(kind), slots=_ints(table[request, place // page] * page + place % page))
        return s
    s.update(q=(2.0 * torch.randn(rows, case["heads"] * dim, generator=generator, device="cuda")).to(torch.bfloat16),
             out=torch.empty(rows, case["heads"] * dim, device="cuda", dtype=torch.bfloat16), table=_ints(table), lengths=_ints(after),
             row_offsets=_ints(np.concatenate([[0], np.cumsum(fresh)])))
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(s):
    return (_CALLS if own else _PLAIN)[s["case"]["path"]](s["case"], s)


# The framework's calls.

def _cache(case, s):
    """The handle of the cache, which a program keeps."""
    from spiraltorch_amd import hip
    if "cache" not in s:
        s["cache"] = hip.KvCache(s["pages"], case["page"], case["kv_heads"], case["dim"], s["k"].data_ptr(), s["v"].data_ptr(),
                                 s["k_scales"].data_ptr(), s["v_scales"].data_ptr())
    return s["cache"]


def _call_tables(case, s):
    from spiraltorch_amd import hip
    hip.page_tables_dev(case["requests"], case["page"], s["cached"].data_ptr(), s["fresh"].data_ptr(), s["free"].numel(), s["free"].data_ptr(),
                        None, s["table"].shape[1], s["table"].data_ptr(), s["rows"], s["row_offsets"].data_ptr(), s["lengths"].data_ptr(),
                        s["positions"].data_ptr(), s["slots"].data_ptr(), s["counts"].data_ptr())
    return {name: s[name] for name in ("table", "row_offsets", "lengths", "positions", "slots", "counts")}


def _rotary(case):
    from spiraltorch_amd import hip
    by_parts = {"original_length": 8192, "low_turns": 1.0, "high_turns": 4.0} if case["by_parts"] else {}
    return hip.Rotary(case["rotary"], base=500000.0, interleaved=case["interleaved"], factor=case["factor"], **by_parts)


def _call_rotary(case, s):
    from spiraltorch_amd import hip
    if "plan" not in s:
        s["plan"] = _rotary(case)
    call = hip.rotary_f32_dev if case["type"] == "f32" else hip.rotary_bf16_dev
    rows, heads, dim = case["rows"], case["heads"], case["dim"]
    call(rows, heads, dim, s["plan"], s["positions"].data_ptr(), s["x"].data_ptr(), case["row_heads"] * dim, s["out"].data_ptr(), heads * dim)
    if not case["gradient"]:
        return s["out"]
    call(rows, heads, dim, s["plan"], s["positions"].data_ptr(), s["g"].data_ptr(), heads * dim, s["gx"].data_ptr(), heads * dim, transposed=True)
    return {"out": s["out"], "gradient": s["gx"]}


def _call_append(case, s):
    from spiraltorch_amd import hip
    call = hip.kv_cache_append_f32_dev if case["type"] == "f32" else hip.kv_cache_append_bf16_dev
    rows, width = s["qkv"].shape
    third = width // 3 * s["qkv"].element_size()
    call(_cache(case, s), rows, s["slots"].data_ptr(), s["qkv"].data_ptr() + third, s["qkv"].data_ptr() + 2 * third, width)
    return {name: s[name] for name in ("k", "v", "k_scales", "v_scales")}


def _call_attention(case, s):
    from spiraltorch_amd import hip
    width = case["heads"] * case["dim"]
    hip.attention_kv_cache_bf16_dev(_cache(case, s), case["requests"], s["q"].shape[0], case["heads"], 1.0 / math.sqrt(case["dim"]),
                                    case["causal"], s["row_offsets"].data_ptr(), s["lengths"].data_ptr(), s["table"].data_ptr(),
                                    s["table"].shape[1], s["q"].data_ptr(), width, s["out"].data_ptr(), width)
    return s["out"]


_CALLS = {"tables": _call_tables, "rotary": _call_rotary, "append": _call_append, "attention": _call_attention}


# The plain forms.

def _plain_tables(case, s):
    page, width, rows = case["page"], s["table"].shape[1], s["rows"]
    cached, fresh = s["cached"].long(), s["fresh"].long()
    ends, after = fresh.cumsum(0), cached + fresh
    had, used = (cached + page - 1) // page, (after + page - 1) // page
    dealt = (used - had).cumsum(0)
    served = (after <= width * page) & (ends <= rows) & ((used == had) | (dealt <= s["free"].numel()))
    column = torch.arange(width, device="cuda")
    new = served[:, None] & (column >= had[:, None]) & (column < used[:, None])
    at = (dealt - used)[:, None] + column  # pages dealt to the requests before, and those of this one before this column
    table = torch.where(new, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"])
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(ends, row, right=True).clamp(max=case["requests"] - 1)
    position = cached[request] + row - (ends - fresh)[request]
    slot = table[request, (position // page).clamp(0, width - 1)].long() * page + position % page
    ok = served[request]
    offsets = torch.cat([ends.new_zeros(1), ends.clamp(max=rows)])
    counts = torch.stack([torch.where(served, used - had, 0).sum(), offsets[-1], (~served).sum()])
    return {"table": table, "row_offsets": offsets.int(), "lengths": torch.where(served, after, 0).int(),
            "positions": torch.where(ok, position, -1).int(), "slots": torch.where(ok, slot, -1).int(), "counts": counts.int()}


def _plain_angles(case, s):
    half = case["rotary"] // 2
    frequency = 500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    if case["by_parts"]:
        kept = ((8192.0 * frequency / (2.0 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        frequency = frequency * (kept + (1.0 - kept) / case["factor"])
    else:
        frequency = frequency / case["factor"]
    angle = s["positions"].double()[:, None, None] * frequency
    return angle.cos().float(), angle.sin().float()


def _plain_turn(case, x, cos, sin):
    x, turned = x.float(), case["rotary"]
    first, second = (x[..., 0:turned:2], x[..., 1:turned:2]) if case["interleaved"] else (x[..., :turned // 2], x[..., turned // 2:turned])
    a, b = first * cos - second * sin, first * sin + second * cos
    both = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([both, x[..., turned:]], -1)


def _plain_rotary(case, s):
    cos, sin = _plain_angles(case, s)
    x = s["x"].view(case["rows"], case["row_heads"], case["dim"])[:, :case["heads"]]
    out = _plain_turn(case, x, cos, sin).to(x.dtype)
    if not case["gradient"]:
        return out
    return {"out": out, "gradient": _plain_turn(case, s["g"], cos, -sin).to(x.dtype)}


def _plain_append(case, s):
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    slots = s["slots"].long()
    touched, at = torch.unique(slots // page, return_inverse=True)
    place = slots % page
    begun = torch.zeros(len(touched), dtype=torch.bool, device="cuda").index_put((at,), place == 0, accumulate=True)
    rows = s["qkv"].float().view(-1, 3, heads, dim)
    for name, x, codes, scales in (("k", rows[:, 1], s["k"], s["k_scales"]), ("v", rows[:, 2], s["v"], s["v_scales"])):
        largest = torch.zeros(len(touched), heads, device="cuda").index_reduce(0, at, x.abs().amax(-1), "amax")
        mantissa, exponent = torch.frexp(largest / LARGEST)  # in 32 bits: the quotient of a value just above 448 * 2^e may round down to 2^e
        needed = torch.ldexp(torch.ones_like(largest), exponent - (mantissa == 0.5).int())
        needed = torch.where(largest > needed * LARGEST, needed * 2.0, needed)
        needed = torch.where(largest > 0, needed, 0.0).clamp(min=SMALLEST_SCALE)
        before = torch.where(begun[:, None], 0.0, scales[touched])
        scale = torch.maximum(before, needed)
        held = codes[touched].float()
        again = torch.where(begun[:, None], 1.0, before / scale)
        held = held * again[:, :, None, None]
        new = x / scale[at][:, :, None]
        if name == "k":
            held[at, :, place] = new
        else:
            held[at, :, :, place] = new
        codes.view(torch.uint8)[touched] = held.to(E4M3).view(torch.uint8)
        scales[touched] = scale
    return {name: s[name] for name in ("k", "v", "k_scales", "v_scales")}


def _plain_attention(case, s):
    page, kv_heads, dim, group, n = case["page"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"], case["requests"]
    fresh, width = case["fresh"], s["table"].shape[1]
    table = s["table"].long().clamp(min=0)
    k = (s["k"].view(torch.uint8)[table].view(E4M3).float() * s["k_scales"][table][..., None, None])
    k = k.permute(0, 2, 1, 3, 4).reshape(n * kv_heads, width * page, dim)
    q = s["q"].float().view(n, fresh, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n * kv_heads, fresh * group, dim)
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).view(n, kv_heads, fresh, group, width * page) / math.sqrt(dim)
    del k
    key = torch.arange(width * page, device="cuda")
    length = s["lengths"].long()[:, None]
    last = length - (fresh - 1 - torch.arange(fresh, device="cuda")) if case["causal"] else length.expand(n, fresh)
    seen = (key < last[..., None]).view(n, 1, fresh, 1, width * page)
    scores = torch.where(seen, scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores - torch.where(most > -math.inf, most, 0.0))
    total = scores.sum(-1, keepdim=True)
    scores = torch.where(seen, scores / torch.where(total > 0, total, 1.0), 0.0).view(n * kv_heads, fresh * group, width * page)
    v = (s["v"].view(torch.uint8)[table].view(E4M3).float() * s["v_scales"][table][..., None, None])
    v = v.permute(0, 2, 1, 4, 3).reshape(n * kv_heads, width * page, dim)
    out = torch.bmm(scores, v).view(n, kv_heads, fresh, group, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(n * fresh, case["heads"] * dim).to(torch.bfloat16)


_PLAIN = {"tables": _plain_tables, "rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    path = case["path"]
    if path == "tables":
        n = case["requests"]
        rows = n - case["prompts"] + case["prompts"] * (case["fresh"] + 1) // 2
        return {"bytes": 4 * (2 * n + 2 * (n + 1) + 2 * rows + 2 * _pages(rows, case["page"])), "flops": 0}
    if path == "rotary":
        values, size = case["rows"] * case["heads"] * case["dim"], 4 if case["type"] == "f32" else 2
        passes = 2 if case["gradient"] else 1
        return {"bytes": passes * (2 * size * values + 4 * case["rows"]), "flops": passes * 3 * values * case["rotary"] // case["dim"]}
    if path == "append":
        rows, size = case["requests"] * case["fresh"], 4 if case["type"] == "f32" else 2
        values = rows * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * values * (size + 1) + 4 * rows, "flops": 4 * values}
    n, low, high, fresh = case["requests"], case["shortest"], case["longest"], case["fresh"]
    length = low if low == high else (high - low) / math.log(high / low)  # on average
    rows = n * fresh
    keys = length if not case["causal"] else max(length - (fresh - 1) / 2, length / 2)  # a row sees, on average
    held = n * length * case["kv_heads"] * (2 * case["dim"] + 8 / case["page"])
    return {"bytes": int(held + 4 * rows * case["heads"] * case["dim"]), "flops": int(4 * rows * keys * case["heads"] * case["dim"])}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["path"]](case, s)


def _exact_tables(case, s):
    page, width, rows = case["page"], s["table"].shape[1], s["rows"]
    cached, fresh, free, table = (s[name].cpu().numpy().astype(np.int64) for name in ("cached", "fresh", "free", "table"))
    offsets, lengths, positions, slots = [0], [], np.full(rows, -1), np.full(rows, -1)
    asked, taken, refused = 0, 0, 0
    for r in range(case["requests"]):
        had, used = -(-cached[r] // page), -(-(cached[r] + fresh[r]) // page)
        first = asked
        asked += used - had
        start = offsets[-1]
        served = used <= width and start + fresh[r] <= rows and (used == had or asked <= len(free))
        offsets.append(min(rows, start + fresh[r]))
        lengths.append(cached[r] + fresh[r] if served else 0)
        refused += not served
        if served:
            table[r, had:used] = free[first:asked]
            taken += used - had
            for i in range(fresh[r]):
                at = cached[r] + i
                positions[start + i], slots[start + i] = at, table[r, at // page] * page + at % page
    return {"table": table, "row_offsets": np.array(offsets), "lengths": np.array(lengths), "positions": positions, "slots": slots,
            "counts": np.array([taken, offsets[-1], refused])}


def _exact_rotary(case, s):
    x, turned = s["x"].double().view(case["rows"], -1, case["dim"])[:, :case["heads"]], case["rotary"]
    pairs = np.arange(turned // 2)
    frequency = np.power(500000.0, -2.0 * pairs / turned)
    slow = frequency / case["factor"]
    if case["by_parts"]:
        kept = np.clip((frequency * 8192 / (2 * np.pi) - 1.0) / (4.0 - 1.0), 0, 1)
        frequency = kept * frequency + (1 - kept) * slow
    else:
        frequency = slow
    turns = torch.polar(torch.ones(case["rows"], 1, turned // 2, device="cuda", dtype=torch.float64),
                        s["positions"].double()[:, None, None] * torch.from_numpy(frequency).cuda())
    first, second = (2 * pairs, 2 * pairs + 1) if case["interleaved"] else (pairs, pairs + turned // 2)

    def turn(values, by):
        out = values.clone()
        z = torch.complex(values[..., first], values[..., second]) * by
        out[..., first], out[..., second] = z.real, z.imag
        return out

    if not case["gradient"]:
        return turn(x, turns)
    return {"out": turn(x, turns), "gradient": turn(s["g"].double(), turns.conj())}


def _exact_append(case, s):
    """Codes as they would be without a last rounding, and the scales."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    slots = s["slots"].cpu().numpy()
    rows = s["qkv"].double().view(-1, 3, heads, dim).cpu().numpy()
    result = {}
    for name, x in (("k", rows[:, 1]), ("v", rows[:, 2])):
        codes = s[name].float().double().cpu().numpy()
        scales = s[name + "_scales"].double().cpu().numpy()
        for p in np.unique(slots // page):
            mine = np.nonzero(slots // page == p)[0]
            places = slots[mine] % page
            largest = np.abs(x[mine]).max(axis=(0, 2))
            needed = np.array([2.0 ** max(-118, math.ceil(math.log2(a) - math.log2(448.0))) if a > 0 else 2.0 ** -118 for a in largest])
            needed = np.where(largest > 448.0 * needed, 2 * needed, np.where(largest <= 224.0 * needed, needed / 2, needed))
            if (places == 0).any():
                scale = needed
            else:
                scale = np.maximum(needed, scales[p])
                codes[p] *= (scales[p] / scale)[:, None, None]
            for place, row in zip(places, mine):
                if name == "k":
                    codes[p, :, place] = x[row] / scale[:, None]
                else:
                    codes[p, :, :, place] = x[row] / scale[:, None]
            scales[p] = scale
        result[name], result[name + "_scales"] = codes, scales
    return result


def _exact_attention(case, s):
    page, group, dim, fresh = case["page"], case["heads"] // case["kv_heads"], case["dim"], case["fresh"]
    out = torch.zeros(s["q"].shape[0], case["heads"], dim, device="cuda", dtype=torch.float64)
    lengths, table = s["lengths"].cpu().numpy(), s["table"].cpu().numpy()
    for r, length in enumerate(lengths):
        used = torch.from_numpy(table[r, :-(-length // page)].astype(np.int64)).cuda()
        q = s["q"][r * fresh:(r + 1) * fresh].double().view(fresh, case["heads"], dim)
        for h in range(case["kv_heads"]):
            k = s["k"].view(torch.uint8)[used, h].view(E4M3).float().double() * s["k_scales"][used, h].double()[:, None, None]
            v = s["v"].view(torch.uint8)[used, h].view(E4M3).float().double() * s["v_scales"][used, h].double()[:, None, None]
            k, v = k.reshape(-1, dim)[:length], v.transpose(1, 2).reshape(-1, dim)[:length]
            mine = q[:, h * group:(h + 1) * group].reshape(fresh * group, dim)
            scores = mine @ k.t() / dim ** 0.5
            if case["causal"]:
                row = torch.arange(fresh, device="cuda").repeat_interleave(group)
                hidden = torch.arange(int(length), device="cuda")[None] > (int(length) - fresh + row)[:, None]
                scores = scores.masked_fill(hidden, -math.inf)
            weights = torch.nan_to_num(torch.softmax(scores, -1))  # a row without keys
            out[r * fresh:(r + 1) * fresh, h * group:(h + 1) * group] = (weights @ v).view(fresh, group, dim)
    return out.view(-1, case["heads"] * dim)


_EXACT = {"tables": _exact_tables, "rotary": _exact_rotary, "append": _exact_append, "attention": _exact_attention}
