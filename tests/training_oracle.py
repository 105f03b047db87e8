"""Attention and its gradients in 64 bits, from the formulas, with how far a kernel may be off that rounds where the contract says.

u = 2^-8 is half a step of bf16, f = 2^-24 of f32.  A sum of n products in f32 is off by at most n f of the sum of their sizes.  The
exponential instruction gives no subnormal numbers: a probability below 2^-126 may come out as 0, which is off by less than LEAST.
"""
import math

import numpy as np

U, F, LEAST = 2.0**-8, 2.0**-24, 2.0**-126


def bucket_of(distance, buckets, max_distance, bidirectional):
    """The bucket of key - query, in whole numbers: bucket e + j begins where m^(s-e) e^j >= far^j e^(s-e)."""
    side, first = buckets, 0
    if bidirectional:
        side //= 2
        first = side if distance > 0 else 0
    m = abs(distance) if bidirectional else max(-distance, 0)
    e = side // 2
    if m < e:
        return first + m
    steps = side - e
    j = max(j for j in range(steps + 1) if m**steps * e**j >= max_distance**j * e**steps)
    return first + min(e + j, side - 1)


def bucket_matrix(n, buckets, max_distance, bidirectional):
    by_distance = np.array([bucket_of(d, buckets, max_distance, bidirectional) for d in range(1 - n, n)])
    at = np.arange(n)
    return by_distance[at[None] - at[:, None] + n - 1]


def head(q, k, v, g, scale, seen, bias, operand, exact_delta=False):
    """One head: (n, d) arrays, seen (n, n) truth values, bias (n, n) or 0.  `operand`: half a step of what p and ds are rounded to for the
    products, 0 for none; results are not rounded.  Returns values and bounds by name."""
    n, d = q.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        s = np.where(seen, scale * (q @ k.T) + bias, -np.inf)
        most = s.max(-1, initial=-np.inf)
        most = np.where(np.isfinite(most), most, 0.0)
        w = np.exp(s - most[:, None])
        total = w.sum(-1)
        lse = most + np.log(total)
        p = w / np.where(total > 0, total, 1.0)[:, None]
    o, dp = p @ v, g @ v.T
    delta = (p * dp).sum(-1)
    ds = p * (dp - delta[:, None])
    abs_ = np.abs
    # the scores: d products, the scale, the bias; in units of log2 e, with as many roundings again for the subtraction and the exponential
    size = np.where(seen, abs_(scale) * (abs_(q) @ abs_(k).T) + np.where(np.isfinite(bias), abs_(bias), 0.0), 0.0)
    e_s = (d + 8) * F * size.max(-1, initial=0.0) + 16 * F * (1 + abs_(np.where(np.isfinite(lse), lse, 0.0)))
    e_lse = e_s + (n + 4) * F
    e_p = (e_s + e_lse)[:, None] + 4 * F  # relative
    e_o = (operand + 2 * e_p + (n + 8) * F) * (p @ abs_(v)) + LEAST * abs_(v).sum(0)
    e_dp = d * F * (abs_(g) @ abs_(v).T)
    if exact_delta:
        e_delta = ((e_p + n * F) * p * abs_(dp) + p * e_dp).sum(-1)
    else:  # of the rounded output
        e_delta = (abs_(g) * (e_o + operand * abs_(o) + d * F * abs_(o))).sum(-1)
    e_ds = abs_(ds) * (e_p + 4 * F) + p * (1 + e_p) * (e_dp + e_delta[:, None]) + LEAST * (1 + abs_(dp) + abs_(delta)[:, None])
    rounded = e_ds + operand * (abs_(ds) + e_ds)
    return {
        "out": (o, e_o), "lse": (lse, e_lse), "ds": (ds, e_ds),
        "dq": (scale * (ds @ k), abs_(scale) * ((rounded + n * F * abs_(ds)) @ abs_(k))),
        "dk": (scale * (ds.T @ q), abs_(scale) * ((rounded + n * F * abs_(ds)).T @ abs_(q))),
        "dv": (p.T @ g, ((operand + e_p + n * F) * p + LEAST).T @ abs_(g)),
    }


def training(q, k, v, g, scale, causal, lengths, table=None, far=0, bidirectional=False):
    """q, g (batch, n, heads, d); k, v (batch, n, kv_heads, d), values of bf16.  Returns {name: (value, bound)} of what the bf16 kernels give."""
    batch, n, heads, d = q.shape
    kv_heads = k.shape[2]
    zero = lambda *shape: [np.zeros(shape), np.zeros(shape)]
    r = {"out": zero(*q.shape), "lse": [np.full((batch, heads, n), -np.inf), np.zeros((batch, heads, n))], "dq": zero(*q.shape), "dk": zero(*k.shape),
         "dv": zero(*k.shape)}
    if table is not None:
        bucket = bucket_matrix(n, table.shape[0], far, bidirectional)
        r["dtable"] = zero(*table.shape)
    for b in range(batch):
        m = n if lengths is None else min(max(int(lengths[b]), 0), n)
        if m == 0:
            continue
        seen = np.tril(np.ones((m, m), bool)) if causal else np.ones((m, m), bool)
        for h in range(heads):
            kv = h * kv_heads // heads
            bias = 0.0 if table is None else table[bucket[:m, :m], h]
            one = head(q[b, :m, h], k[b, :m, kv], v[b, :m, kv], g[b, :m, h], scale, seen, bias, U, exact_delta=False)
            for i in (0, 1):
                r["out"][i][b, :m, h] = one["out"][i]
                r["lse"][i][b, h, :m] = one["lse"][i]
                r["dq"][i][b, :m, h] = one["dq"][i]
                r["dk"][i][b, :m, kv] += one["dk"][i]
                r["dv"][i][b, :m, kv] += one["dv"][i]
            if table is not None:
                ds, e_ds = head(q[b, :m, h], k[b, :m, kv], v[b, :m, kv], g[b, :m, h], scale, seen, bias, U, exact_delta=True)["ds"]
                for c in range(table.shape[0]):
                    mine = bucket[:m, :m] == c
                    r["dtable"][0][c, h] += ds[mine].sum()
                    r["dtable"][1][c, h] += (e_ds[mine] + (m + batch * m) * F * np.abs(ds[mine])).sum()
    for name in ("out", "dq", "dk", "dv"):
        value, bound = r[name]
        r[name] = (value, bound + U * (np.abs(value) + bound) + 2.0**-133)  # stored in bf16
    return r


def check(got, want, what):
    """want: (value, bound).  Infinities have to be where they are."""
    value, bound = want
    got = np.asarray(got, np.float64).reshape(value.shape)
    same = (got == value)
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - value))
    assert not np.isnan(off).any(), f"{what}: {np.isnan(off).sum()} of {off.size} are NaN"
    bad = off > np.where(np.isfinite(value), bound, 0.0)
    if math.prod(off.shape) and bad.any():
        at = np.unravel_index(int(np.argmax(np.where(bad, off - bound, -1))), off.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; at {at}: {got[at]!r} for {value[at]!r}, off by {off[at]:.3e}, bound {bound[at]:.3e}")
