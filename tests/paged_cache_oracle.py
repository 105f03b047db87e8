"""Plain forms, in 64 bits on the CPU, of the operators around the paged 8-bit cache."""
import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


def widen(codes):
    """e4m3 bytes -> float64."""
    return torch.from_numpy(np.ascontiguousarray(codes)).view(E4M3).to(torch.float64).numpy()


def narrow(values):
    """Values that are at most 448 in size, or NaN -> e4m3 bytes, to nearest, ties to even (all of them exact in f32, or far from a tie)."""
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.float32)).to(E4M3).view(torch.uint8).numpy()


def page_tables(page, cached, fresh, free_pages, taken_before, table, rows):
    """row_offsets, lengths, positions, slots, counts and the table afterwards."""
    requests, width = table.shape
    table = table.copy()
    offsets, lengths = [0], []
    positions, slots = [-1] * rows, [-1] * rows
    pages_of = lambda tokens: -(-tokens // page)
    asked, taken, refused, start = 0, 0, 0, 0
    left = max(0, len(free_pages) - taken_before)
    for r in range(requests):
        c, f = int(cached[r]), int(fresh[r])
        mine = max(0, f)
        possible = c >= 0 and f >= 0 and pages_of(c + f) <= width and c + f <= 2**31 - 1
        need = pages_of(c + f) - pages_of(c) if possible else 0
        first = taken_before + asked
        asked += need
        served = possible and start + mine <= rows and (need == 0 or asked <= left)
        if served:
            taken += need
            table[r, pages_of(c):pages_of(c) + need] = free_pages[first:first + need]
        else:
            refused += 1
        for i in range(mine):
            if start + i >= rows:
                break
            if served:
                positions[start + i] = c + i
                at = int(table[r, (c + i) // page])
                slot = at * page + (c + i) % page
                slots[start + i] = slot if at >= 0 and slot <= 2**31 - 1 else -1
        start += mine
        offsets.append(min(start, rows))
        lengths.append(c + f if served else 0)
    return offsets, lengths, positions, slots, [taken_before + taken, min(start, rows), refused], table


def turns(rotary_dim, base=10000.0, factor=1.0, original_length=0.0, low_turns=1.0, high_turns=4.0):
    """Radians that each pair turns per position."""
    plain = base ** (-2.0 * np.arange(rotary_dim // 2) / max(1, rotary_dim))
    if original_length <= 0:
        return plain / factor
    kept = np.clip((original_length * plain / (2 * np.pi) - low_turns) / (high_turns - low_turns), 0, 1)
    return plain * (kept + (1 - kept) / factor)


def rotary(x, positions, rotary_dim, interleaved, per_position, magnitude=1.0, transposed=False):
    """x (rows, heads, head_dim) -> the same, turned; and for every value the sum of the sizes that its products have."""
    half = rotary_dim // 2
    first = 2 * np.arange(half) if interleaved else np.arange(half)
    second = first + (1 if interleaved else half)
    angle = np.asarray(positions, np.float64)[:, None, None] * per_position
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if transposed else 1)
    out, size = x.astype(np.float64).copy(), np.zeros(x.shape)
    a, b = out[..., first].copy(), out[..., second].copy()
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = (np.abs(a) + np.abs(b)) * abs(magnitude)
    return out, size


def needed_scale(largest):
    scale = 2.0 ** -118
    while largest > 448.0 * scale:
        scale *= 2.0
    return scale


def append(codes, scales, slots, rows, transposed):
    """codes (pages, heads, page, dim), or (pages, heads, dim, page) if `transposed`, with scales (pages, heads): the rows
    (n, heads, dim) put in, in place."""
    page = codes.shape[3 if transposed else 2]
    pages = codes.shape[0]
    by_page = {}
    for i, slot in enumerate(slots):
        if 0 <= slot < pages * page:
            by_page.setdefault(int(slot) // page, {})[int(slot) % page] = i
    for p, places in by_page.items():
        for h in range(codes.shape[1]):
            block = codes[p, h].T if transposed else codes[p, h]  # (page, dim), a view
            new = {place: rows[i, h].astype(np.float64) for place, i in places.items()}
            every = np.concatenate(list(new.values()))
            every = np.abs(every[np.isfinite(every)])
            scale = needed_scale(every.max() if every.size else 0.0)
            if 0 not in places:
                scale = max(scale, float(scales[p, h]))
                if scale > scales[p, h]:
                    others = [t for t in range(page) if t not in places]
                    block[others] = narrow(widen(block[others]) * (float(scales[p, h]) / scale))
            scales[p, h] = scale
            for place, x in new.items():
                y = x / scale
                block[place] = narrow(np.where(np.abs(y) <= 448.0, y, np.nan))


def attention(k, v, k_scales, v_scales, offsets, lengths, table, q, scale, causal, weight_step=2.0**-8):
    """k (pages, heads, page, dim), v (pages, heads, dim, page) codes; q (rows, heads, dim) float64.  The result, the rows that belong to
    a request, and how far a result may be off that is computed as the kernel does it:

      a score is a sum of head_dim products in f32 in any order, times two scales and log2(e): (head_dim + 4) half steps of the sum of
      the sizes, and one more for the difference to the maximum; a weight carries twice that, as the largest score shifts all of them;
      its power of two a few steps; weights are rounded to bf16 (2^-8 of each, or weight_step where they are in pieces), in the sum of the weights as in that of the values: a
      result sum(w v) / sum(w) moves by sum(dw (v - result)) / sum(w); both are summed in f32 (a half step per key at the most), and
      the result is rounded to bf16."""
    rows, heads, dim = q.shape
    pages, kv_heads, page = k.shape[:3]
    group = heads // kv_heads
    out, mine, bound = np.zeros((rows, heads, dim)), np.zeros(rows, bool), np.zeros((rows, heads, dim))
    for r, length in enumerate(lengths):
        first, end = offsets[r], offsets[r + 1]
        mine[first:end] = True
        length = min(max(0, int(length)), table.shape[1] * page)
        used = table[r, :-(-length // page)]
        there = np.repeat((used >= 0) & (used < pages), page)[:length]
        safe = np.where((used >= 0) & (used < pages), used, 0)
        for h in range(kv_heads):
            keys = (widen(k[safe, h]) * k_scales[safe, h, None, None].astype(np.float64)).reshape(-1, dim)[:length]
            values = (widen(v[safe, h]) * v_scales[safe, h, None, None].astype(np.float64)).transpose(0, 2, 1).reshape(-1, dim)[:length]
            for i in range(first, end):
                seen = there & (np.arange(length) <= length - (end - i) if causal else True)
                if not seen.any():
                    continue
                for head in range(h * group, (h + 1) * group):
                    x = q[i, head]
                    with np.errstate(all="ignore"):
                        scores = keys[seen] @ x * scale
                        weights = np.exp(scores - scores.max())
                        total = weights.sum()
                        out[i, head] = weights @ values[seen] / total
                        sizes = (weights @ np.abs(values[seen])) / total
                        off = (dim + 8) * 2.0**-24 * np.max(np.abs(keys[seen]) @ np.abs(x)) * abs(scale)
                    weights_off = weight_step * 1.01 + 4 * off + (8 + seen.sum()) * 2.0**-24
                    bound[i, head] = 2.0**-8 * np.abs(out[i, head]) + weights_off * (sizes + np.abs(out[i, head]))
    return out, mine, bound
