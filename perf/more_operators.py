"""Training a decoder and scoring what it says: the operators, their plain forms and the work they are asked for.

Three paths: `attention` (bf16 attention that is trained: its forward pass with the log-sum-exp kept and its backward pass, heads that share
keys, padded batches, a learned bias by buckets of distance with the table's gradient), `attention_f32` (the backward pass of the f32
attention with additive biases, and theirs) and `log_probs` (log-probabilities of given tokens, entropies, the likeliest alternatives,
and the gradient of the logits).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # A short batch, forward and backward: latency.
        {"name": "attention_3x37", "path": "attention", "batch": 3, "heads": 4, "kv_heads": 4, "sequence": 37, "dim": 64, "causal": True,
         "shortest": 37, "buckets": 0, "farthest": 0},
        # The byte-level decoder's batch: 16 x 1024 tokens, 8 heads of 64.
        {"name": "attention_16x1024", "path": "attention", "batch": 16, "heads": 8, "kv_heads": 8, "sequence": 1024, "dim": 64, "causal": True,
         "shortest": 1024, "buckets": 0, "farthest": 0},
        # One long document, four heads of queries on each of keys.
        {"name": "attention_1x8192_shared", "path": "attention", "batch": 1, "heads": 32, "kv_heads": 8, "sequence": 8192, "dim": 128,
         "causal": True, "shortest": 8192, "buckets": 0, "farthest": 0},
        # An encoder's padded batch, all lengths.
        {"name": "attention_8x1500_padded", "path": "attention", "batch": 8, "heads": 12, "kv_heads": 12, "sequence": 1500, "dim": 64,
         "causal": False, "shortest": 90, "buckets": 0, "farthest": 0},
        # An encoder with positions learned by buckets of distance.
        {"name": "attention_16x512_buckets", "path": "attention", "batch": 16, "heads": 12, "kv_heads": 12, "sequence": 512, "dim": 64,
         "causal": False, "shortest": 200, "buckets": 32, "farthest": 128},
        # A decoder with them.
        {"name": "attention_2x2048_buckets", "path": "attention", "batch": 2, "heads": 16, "kv_heads": 4, "sequence": 2048, "dim": 128,
         "causal": True, "shortest": 2048, "buckets": 32, "farthest": 128},
        # The f32 attention's gradients, its biases' among them.
        {"name": "attention_f32_16x1024_biased", "path": "attention_f32", "contexts": 16, "sequence": 1024, "dim": 64, "causal": False,
         "biased": True},
        # Odd sizes, causal, without biases.
        {"name": "attention_f32_96x333", "path": "attention_f32", "contexts": 96, "sequence": 333, "dim": 80, "causal": True, "biased": False},
        # What a decode step's tokens were worth, for one user and for 64, with the likeliest alternatives; a tenth of the vocabulary is barred.
        {"name": "log_probs_1x131072", "path": "log_probs", "rows": 1, "vocab": 131072, "type": "bf16", "top": 20, "barred": 0.1,
         "gradient": False},
        {"name": "log_probs_64x100001", "path": "log_probs", "rows": 64, "vocab": 100001, "type": "f32", "top": 5, "barred": 0.1,
         "gradient": False},
        # The byte-level decoder's loss: 16 x 1024 tokens.
        {"name": "log_probs_16384x256", "path": "log_probs", "rows": 16384, "vocab": 256, "type": "f32", "top": 0, "barred": 0.0,
         "gradient": True},
        # A loss with an entropy term over a large odd vocabulary.
        {"name": "log_probs_8192x50001", "path": "log_probs", "rows": 8192, "vocab": 50001, "type": "bf16", "top": 0, "barred": 0.0,
         "gradient": True},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    path = rng.choice(["attention", "attention", "attention", "attention_f32", "log_probs", "log_probs"])
    most = {key: max(work(case)[key] for case in listed() if case["path"] == path) for key in ("bytes", "flops")}
    while True:
        case = {"path": path}
        if path == "attention":
            kv_heads, sequence, buckets = _log(rng, 1, 16), _log(rng, 1, 8192), rng.choice([0, 0, 8, 32, 64])
            case.update(batch=_log(rng, 1, 32), heads=kv_heads * rng.choice([1, 1, 2, 4, 7]), kv_heads=kv_heads, sequence=sequence,
                        dim=rng.choice([64, 64, 128]), causal=rng.random() < 0.6, shortest=rng.choice([sequence, _log(rng, 1, sequence)]),
                        buckets=buckets, farthest=rng.choice([64, 128, 300]) if buckets else 0)
            if case["batch"] * case["heads"] * sequence * sequence > 2.2e9:  # what the plain form holds of scores
                continue
        elif path == "attention_f32":
            case.update(contexts=_log(rng, 1, 128), sequence=_log(rng, 1, 2048), dim=rng.choice([8, 32, 64, 80, 128, 256]),
                        causal=rng.random() < 0.5, biased=rng.random() < 0.5)
        else:
            case.update(rows=_log(rng, 1, 16384), vocab=_log(rng, 2, 262144), type=rng.choice(["bf16", "f32"]), top=rng.choice([0, 1, 5, 20]),
                        barred=rng.choice([0.0, 0.1]), gradient=rng.random() < 0.5)
            case["top"] = min(case["top"], case["vocab"] // 2)
            if case["rows"] * case["vocab"] > 4.1e8 or (case["top"] and case["rows"] * case["vocab"] > 3e7):  # the plain form sorts whole rows
                continue
        cost = work(case)
        if cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]:
            return case


# ---- inputs -------------------------------------------------------------------------------------------------------------------

def _lengths(case, seed):
    """The lengths of a padded batch, evenly spread, in an order of the seed."""
    return np.random.default_rng(seed).permutation(np.linspace(case["shortest"], case["sequence"], case["batch"]).astype(np.int64))


def prepare(case, seed):
    s = {"case": case}
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=generator, device="cuda")
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, device="cuda", dtype=dtype)
    if case["path"] == "attention":
        # Queries, keys and values stand in the rows of one projection, and their gradients in those of its gradient.
        rows, dim, width = case["batch"] * case["sequence"], case["dim"], case["heads"] * case["dim"]
        fused = (case["heads"] + 2 * case["kv_heads"]) * dim
        s.update(qkv=normal(rows, fused).to(torch.bfloat16), g=normal(rows, width).to(torch.bfloat16),
                 lengths=torch.tensor(_lengths(case, seed), dtype=torch.int32, device="cuda"),
                 out=empty(rows, width, dtype=torch.bfloat16), lse=empty(case["batch"], case["heads"], case["sequence"]),
                 g_qkv=empty(rows, fused, dtype=torch.bfloat16))
        if case["buckets"]:
            s.update(table=normal(case["buckets"], case["heads"]), g_table=empty(case["buckets"], case["heads"]))
    elif case["path"] == "attention_f32":
        contexts, n, dim = case["contexts"], case["sequence"], case["dim"]
        s.update({name: normal(contexts, n, dim) for name in ("q", "k", "v", "g")})
        s.update({"g_" + name: empty(contexts, n, dim) for name in ("q", "k", "v")})
        if case["biased"]:
            s.update(z=normal(contexts, n), bias=normal(contexts, n, n), g_z=empty(contexts, n), g_bias=empty(contexts, n, n))
        s["out"] = _plain_f32_forward(case, s)[1]  # what the forward pass gave
    else:
        rows, vocab = case["rows"], case["vocab"]
        kind = torch.bfloat16 if case["type"] == "bf16" else torch.float32
        logits = 2.0 * normal(rows, vocab)
        draws = torch.rand(rows, generator=generator, device="cuda")
        tokens = (draws * draws * vocab).int().clamp(max=vocab - 1)  # low ones more often
        logits[torch.arange(rows, device="cuda"), tokens.long()] += 6.0
        if case["barred"]:
            barred = torch.rand(vocab, generator=generator, device="cuda") < case["barred"]
            barred[tokens.long()] = False  # what has been said was allowed
            logits[:, barred] = -math.inf
        tokens[3::17] = -1  # rows that do not count
        s.update(logits=logits.to(kind), tokens=tokens, log_probs=empty(rows), entropies=empty(rows), lse=empty(rows),
                 top_ids=empty(rows, case["top"], dtype=torch.int32), top_log_probs=empty(rows, case["top"]))
        if case["gradient"]:
            s.update(g=normal(rows) / rows, g_entropies=normal(rows) / rows, g_logits=empty(rows, vocab, dtype=kind))
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(s):
    return (_CALLS if own else _PLAIN)[s["case"]["path"]](s["case"], s)


# The framework's calls.

def _call_attention(case, s):
    from spiraltorch_amd import hip
    heads, kv_heads, dim, width, fused = case["heads"], case["kv_heads"], case["dim"], s["out"].shape[1], s["qkv"].shape[1]
    if "plan" not in s:  # a program keeps it
        bias = hip.PositionBias(case["buckets"], case["farthest"], s["table"].data_ptr(), bidirectional=not case["causal"]) if case["buckets"] else None
        s["plan"] = hip.AttentionTraining(case["batch"], heads, case["sequence"], dim, 1.0 / math.sqrt(dim), causal=case["causal"],
                                          kv_heads=kv_heads, lengths=s["lengths"].data_ptr(), position_bias=bias)
    q, gq = s["qkv"].data_ptr(), s["g_qkv"].data_ptr()
    behind_q, behind_k = 2 * width, 2 * (width + kv_heads * dim)
    hip.attention_training_bf16_dev(s["plan"], q, fused, q + behind_q, q + behind_k, fused, s["out"].data_ptr(), width, s["lse"].data_ptr())
    hip.attention_backward_bf16_dev(s["plan"], q, fused, q + behind_q, q + behind_k, fused, s["out"].data_ptr(), width, s["lse"].data_ptr(),
                                    s["g"].data_ptr(), width, gq, fused, gq + behind_q, gq + behind_k, fused,
                                    s["g_table"].data_ptr() if case["buckets"] else None)
    return {name: s[name] for name in ("out", "lse", "g_qkv", "g_table") if name in s}


def _call_attention_f32(case, s):
    from spiraltorch_amd import hip
    at = lambda name: s[name].data_ptr() if name in s else None
    hip.attention_backward_f32_dev(case["contexts"], case["sequence"], case["dim"], 1.0 / math.sqrt(case["dim"]), case["causal"], at("q"), at("k"),
                                   at("v"), at("z"), at("bias"), at("out"), at("g"), at("g_q"), at("g_k"), at("g_v"), at("g_z"), at("g_bias"))
    return {name: s[name] for name in ("g_q", "g_k", "g_v", "g_z", "g_bias") if name in s}


def _call_log_probs(case, s):
    from spiraltorch_amd import hip
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    forward, backward = (hip.token_log_probs_f32_dev, hip.token_log_probs_backward_f32_dev) if case["type"] == "f32" else \
        (hip.token_log_probs_bf16_dev, hip.token_log_probs_backward_bf16_dev)
    at = lambda name: s[name].data_ptr()
    forward(rows, vocab, at("logits"), vocab, at("tokens"), at("log_probs"), at("entropies"), at("lse"), top, at("top_ids"), at("top_log_probs"))
    result = {name: s[name] for name in ("log_probs", "entropies", "lse")}
    if top:
        result.update(top_ids=s["top_ids"], top_log_probs=s["top_log_probs"])
    if case["gradient"]:
        backward(rows, vocab, at("logits"), vocab, at("tokens"), at("lse"), at("entropies"), at("g"), at("g_entropies"), at("g_logits"), vocab)
        result["g_logits"] = s["g_logits"]
    return result


_CALLS = {"attention": _call_attention, "attention_f32": _call_attention_f32, "log_probs": _call_log_probs}


# The plain forms.

def _plain_buckets(case):
    """The bucket of every (query, key)."""
    at = torch.arange(case["sequence"], device="cuda")
    apart = at[None] - at[:, None]
    if case["causal"]:
        half, first, apart = case["buckets"], torch.zeros_like(apart), (-apart).clamp(min=0)
    else:
        half = case["buckets"] // 2
        first, apart = (apart > 0).long() * half, apart.abs()
    exact = half // 2
    far = (half - exact) * torch.log(apart.clamp(min=1).double() / exact) / math.log(case["farthest"] / exact)
    return first + torch.where(apart < exact, apart, (exact + torch.floor(far + 1e-9).long()).clamp(max=half - 1))


def _plain_split(case, qkv):
    """(batch, kv_heads, heads that share them, sequence, dim) of the queries, and so of the keys and values."""
    n, kv_heads, dim, group = case["sequence"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    q, k, v = qkv.split([case["heads"] * dim, kv_heads * dim, kv_heads * dim], 1)
    part = lambda x, m: x.float().view(case["batch"], n, kv_heads, m, dim).permute(0, 2, 3, 1, 4).contiguous()
    return part(q, group), part(k, 1), part(v, 1)


def _plain_joined(case, x):
    return x.permute(0, 3, 1, 2, 4).reshape(case["batch"] * case["sequence"], -1)


def _plain_attention(case, s):
    n, scale = case["sequence"], 1.0 / math.sqrt(case["dim"])
    q, k, v = _plain_split(case, s["qkv"])
    g = s["g"].float().view(case["batch"], n, case["kv_heads"], -1, case["dim"]).permute(0, 2, 3, 1, 4).contiguous()
    at, length = torch.arange(n, device="cuda"), s["lengths"].long()[:, None, None, None, None]
    seen = (at[:, None] < length) & (at < length)
    if case["causal"]:
        seen = seen & (at <= at[:, None])
    flat = lambda x: x.expand(-1, -1, q.shape[2], -1, -1).contiguous()
    scores = torch.matmul(q, flat(k).transpose(-1, -2).contiguous()) * scale
    if case["buckets"]:
        bucket = _plain_buckets(case)
        scores += s["table"][bucket].permute(2, 0, 1).reshape(case["kv_heads"], -1, n, n)
    scores = torch.where(seen, scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most > -math.inf, most, 0.0)
    weights = torch.exp(scores - most)
    del scores
    total = weights.sum(-1, keepdim=True)
    lse = (most + torch.log(total)).view(case["batch"], case["heads"], n)
    weights /= torch.where(total > 0, total, 1.0)
    out = torch.matmul(weights, flat(v))
    grad_v = torch.matmul(weights.transpose(-1, -2).contiguous(), g).sum(2, keepdim=True)
    grad = torch.matmul(g, flat(v).transpose(-1, -2).contiguous())
    grad = weights * (grad - (g * out).sum(-1, keepdim=True))
    del weights
    grad_q = torch.matmul(grad, flat(k)) * scale
    grad_k = torch.matmul(grad.transpose(-1, -2).contiguous(), q).sum(2, keepdim=True) * scale
    result = {"out": _plain_joined(case, out).to(torch.bfloat16), "lse": lse,
              "g_qkv": torch.cat([_plain_joined(case, x) for x in (grad_q, grad_k, grad_v)], 1).to(torch.bfloat16)}
    if case["buckets"]:
        grad = grad.sum(0, dtype=torch.float64).view(-1, n, n)
        result["g_table"] = torch.stack([torch.where(bucket == b, grad, 0.0).sum((1, 2)) for b in range(case["buckets"])]).float()
    return result


def _plain_f32_forward(case, s):
    n = case["sequence"]
    scores = torch.matmul(s["q"], s["k"].transpose(-1, -2).contiguous()) / math.sqrt(case["dim"])
    if case["biased"]:
        scores = scores + s["z"][:, None] + s["bias"]
    if case["causal"]:
        at = torch.arange(n, device="cuda")
        scores = torch.where(at <= at[:, None], scores, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    return weights, torch.matmul(weights, s["v"])


def _plain_attention_f32(case, s):
    weights, out = _plain_f32_forward(case, s)
    grad = torch.matmul(s["g"], s["v"].transpose(-1, -2).contiguous())
    grad = weights * (grad - (s["g"] * out).sum(-1, keepdim=True))
    scale = 1.0 / math.sqrt(case["dim"])
    result = {"g_q": torch.matmul(grad, s["k"]) * scale, "g_k": torch.matmul(grad.transpose(-1, -2).contiguous(), s["q"]) * scale,
              "g_v": torch.matmul(weights.transpose(-1, -2).contiguous(), s["g"])}
    if case["biased"]:
        result.update(g_z=grad.sum(1), g_bias=grad)
    return result


def _plain_log_probs(case, s):
    x = s["logits"].float()
    most = x.amax(-1, keepdim=True)
    lse = most + torch.log(torch.exp(x - most).sum(-1, keepdim=True))
    log_p = x - lse
    p = torch.exp(log_p)
    entropies = -torch.where(p > 0, p * log_p, 0.0).sum(-1)
    counted, token = s["tokens"] >= 0, s["tokens"].long().clamp(min=0)[:, None]
    log_probs = torch.where(counted, log_p.gather(1, token)[:, 0], 0.0)
    result = {"log_probs": log_probs, "entropies": entropies, "lse": lse[:, 0]}
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]]  # the lowest of equal ones first
        result.update(top_ids=ids.int(), top_log_probs=log_p.gather(1, ids))
    if case["gradient"]:
        g = torch.where(counted, s["g"], 0.0)[:, None]
        gradient = -g * p - s["g_entropies"][:, None] * torch.where(p > 0, p * (log_p + entropies[:, None]), 0.0)
        result["g_logits"] = gradient.scatter_add_(1, token, g).to(s["logits"].dtype)
    return result


_PLAIN = {"attention": _plain_attention, "attention_f32": _plain_attention_f32, "log_probs": _plain_log_probs}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    if case["path"] == "attention":
        lengths = np.linspace(case["shortest"], case["sequence"], case["batch"]).astype(np.int64).astype(float)
        pairs = float((lengths * (lengths + 1) / 2 if case["causal"] else lengths * lengths).sum()) * case["heads"]
        tokens, heads, kv_heads = float(lengths.sum()), case["heads"], case["kv_heads"]
        # q, k, v and the output's gradient in, the output, the log-sum-exp and three gradients out
        moved = tokens * (2 * case["dim"] * (4 * heads + 4 * kv_heads) + 4 * heads) + 8 * case["buckets"] * heads
        return {"bytes": int(moved), "flops": int(14 * pairs * case["dim"])}  # two products, and five more of the backward pass
    if case["path"] == "attention_f32":
        n, contexts = case["sequence"], case["contexts"]
        pairs = contexts * (n * (n + 1) // 2 if case["causal"] else n * n)
        biases = 8 * contexts * (n + n * n) if case["biased"] else 0
        return {"bytes": 4 * contexts * n * case["dim"] * 8 + biases, "flops": 10 * pairs * case["dim"]}
    values, size = case["rows"] * case["vocab"], 2 if case["type"] == "bf16" else 4
    return {"bytes": values * size * (3 if case["gradient"] else 1) + case["rows"] * (16 + 8 * case["top"]),
            "flops": values * (12 if case["gradient"] else 6)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    return _EXACT[case["path"]](case, prepare(case, seed))


def _exact_bucket(case, apart):
    """The bucket of a key `apart` behind its query, in whole numbers: m >= exact * (farthest / exact)^(j / steps) for the j-th one."""
    half, first = case["buckets"], 0
    if not case["causal"]:
        half //= 2
        first = half if apart > 0 else 0
    m = max(-apart, 0) if case["causal"] else abs(apart)
    exact, far = half // 2, case["farthest"]
    if m < exact:
        return first + m
    steps = half - exact
    j = max(j for j in range(steps + 1) if m ** steps * exact ** j >= far ** j * exact ** steps)
    return first + min(exact + j, half - 1)


def _exact_attention(case, s):
    batch, n, heads, kv_heads, dim = case["batch"], case["sequence"], case["heads"], case["kv_heads"], case["dim"]
    qkv, g = s["qkv"].view(batch, n, heads + 2 * kv_heads, dim), s["g"].view(batch, n, heads, dim)
    zeros = lambda *shape: torch.zeros(*shape, device="cuda", dtype=torch.float64)
    out, lse, g_qkv = zeros(batch, n, heads, dim), torch.full_like(s["lse"], -math.inf, dtype=torch.float64), zeros(*qkv.shape)
    if case["buckets"]:
        by_distance = torch.tensor([_exact_bucket(case, d) for d in range(1 - n, n)], device="cuda")
        at = torch.arange(n, device="cuda")
        bucket = by_distance[at[None] - at[:, None] + n - 1]
        g_table = zeros(case["buckets"], heads)
    for b, length in enumerate(s["lengths"].tolist()):
        for h in range(heads):
            mine = [h, heads + h * kv_heads // heads, heads + kv_heads + h * kv_heads // heads]
            q, k, v = (qkv[b, :length, i].double().requires_grad_() for i in mine)
            scores = q @ k.t() / dim ** 0.5
            if case["buckets"]:
                column = s["table"][:, h].double().requires_grad_()
                # (one product with what chooses the bucket: an indexed gradient would be added value by value)
                scores = scores + sum(column[c] * (bucket[:length, :length] == c) for c in range(case["buckets"]))
            if case["causal"]:
                scores = scores.masked_fill(torch.ones(length, length, device="cuda", dtype=torch.bool).triu(1), -math.inf)
            lse[b, h, :length] = torch.logsumexp(scores.detach(), -1)
            o = torch.softmax(scores, -1) @ v
            o.backward(g[b, :length, h].double())
            out[b, :length, h] = o.detach()
            for i, x in zip(mine, (q, k, v)):
                g_qkv[b, :length, i] += x.grad
            if case["buckets"]:
                g_table[:, h] += column.grad
    result = {"out": out.view(batch * n, -1), "lse": lse, "g_qkv": g_qkv.view(batch * n, -1)}
    if case["buckets"]:
        result["g_table"] = g_table
    return result


def _exact_attention_f32(case, s):
    names = ["q", "k", "v"] + (["z", "bias"] if case["biased"] else [])
    gradients = {name: [] for name in names}
    for c in range(case["contexts"]):
        x = {name: s[name][c].double().requires_grad_() for name in names}
        scores = x["q"] @ x["k"].t() / case["dim"] ** 0.5
        if case["biased"]:
            scores = scores + x["z"] + x["bias"]
        if case["causal"]:
            scores = scores.masked_fill(torch.ones_like(scores, dtype=torch.bool).triu(1), -math.inf)
        (torch.softmax(scores, -1) @ x["v"]).backward(s["g"][c].double())
        for name in names:
            gradients[name].append(x[name].grad)
    return {"g_" + name: torch.stack(gradients[name]) for name in names}


def _exact_log_probs(case, s):
    x, rows = s["logits"].double(), case["rows"]
    counted, token = s["tokens"] >= 0, s["tokens"].long().clamp(min=0)
    lse = torch.logsumexp(x, -1)
    p = torch.softmax(x, -1)
    entropies = torch.special.entr(p).sum(-1)
    row = torch.arange(rows, device="cuda")
    result = {"log_probs": torch.where(counted, x[row, token] - lse, 0.0), "entropies": entropies, "lse": lse}
    if case["top"]:
        ids = np.argsort(-x.cpu().numpy(), -1, kind="stable")[:, :case["top"]]
        result.update(top_ids=ids, top_log_probs=torch.log(p.gather(1, torch.from_numpy(ids).cuda())))
    if case["gradient"]:
        one = torch.zeros_like(x)
        one[row, token] = 1.0
        d = (one - p) * torch.where(counted, s["g"].double(), 0.0)[:, None]
        result["g_logits"] = d + s["g_entropies"].double()[:, None] * (torch.special.entr(p) - p * entropies[:, None])
    return result


_EXACT = {"attention": _exact_attention, "attention_f32": _exact_attention_f32, "log_probs": _exact_log_probs}
