"""The paged 8-bit cache on the GPU: page tables, appending, attention over it, and a run of them together."""
import numpy as np
import pytest

import paged_cache_oracle as plain
from spiraltorch_amd import inputs

pytestmark = pytest.mark.gpu

SENTINEL = -77


def dev(hip, array, dtype=np.int32):
    return hip.DeviceBuffer.from_array(np.ascontiguousarray(array, dtype=dtype))


# ---- page tables ----------------------------------------------------------------------------------------------------------------

def check_tables(hip, page, cached, fresh, free_pages, taken_before, table, rows):
    requests, width = table.shape
    bufs = {"cached": dev(hip, cached), "fresh": dev(hip, fresh), "free": dev(hip, free_pages) if len(free_pages) else None,
            "before": None if taken_before is None else dev(hip, [taken_before]), "table": dev(hip, table) if table.size else None,
            "offsets": dev(hip, np.full(requests + 3, SENTINEL)), "lengths": dev(hip, np.full(requests + 2, SENTINEL)),
            "positions": dev(hip, np.full(rows + 5, SENTINEL)), "slots": dev(hip, np.full(rows + 5, SENTINEL)), "counts": dev(hip, [SENTINEL] * 4)}
    hip.page_tables_dev(requests, page, bufs["cached"], bufs["fresh"], len(free_pages), bufs["free"], bufs["before"], width, bufs["table"], rows,
                        bufs["offsets"], bufs["lengths"], bufs["positions"], bufs["slots"], bufs["counts"])
    hip.device_synchronize()
    offsets, lengths, positions, slots, counts, after = plain.page_tables(page, cached, fresh, free_pages, max(0, taken_before or 0), table, rows)
    read = lambda name, n: bufs[name].to_array(np.int32, n).tolist()
    assert read("offsets", requests + 3) == offsets + [SENTINEL] * 2
    assert read("lengths", requests + 2) == lengths + [SENTINEL] * 2
    assert read("positions", rows + 5) == positions + [SENTINEL] * 5
    assert read("slots", rows + 5) == slots + [SENTINEL] * 5
    assert read("counts", 4) == counts + [SENTINEL]
    if table.size:
        assert (bufs["table"].to_array(np.int32, table.shape) == after).all()


def make_tables(rng, requests, page, longest, fresh_most, spare=3, width=None):
    cached, fresh = rng.integers(0, longest + 1, requests), rng.integers(0, fresh_most + 1, requests)
    had = -(-cached // page)
    width = width or int(-(-(longest + fresh_most) // page)) + 1
    order = rng.permutation(int(had.sum()) + int((-(-(cached + fresh) // page) - had).sum()) + spare)
    table, at = np.full((requests, width), SENTINEL), 0
    for r in range(requests):
        table[r, :had[r]] = order[at:at + had[r]]
        at += had[r]
    return cached, fresh, order[at:], table


@pytest.mark.parametrize("requests,page,longest,fresh", [(1, 16, 0, 1), (1, 64, 100, 1), (1, 256, 4000, 3000), (2, 16, 40, 16), (7, 32, 300, 200),
                                                        (64, 64, 4096, 1), (255, 128, 500, 40), (257, 16, 90, 33), (1023, 16, 60, 3),
                                                        (1025, 32, 50, 9), (2100, 64, 200, 5), (3, 16, 10, 5000)])
def test_tables(hip, requests, page, longest, fresh):
    rng = np.random.default_rng(requests + page)
    cached, new, free, table = make_tables(rng, requests, page, longest, fresh)
    rows = int(new.sum())
    check_tables(hip, page, cached, new, free, None, table, rows)
    check_tables(hip, page, cached, new, np.concatenate([[9, 9], free]), 2, table, rows + 1500)  # taken before, and room behind the rows


def test_tables_of_nothing(hip):
    check_tables(hip, 64, [], [], [1, 2], 1, np.zeros((0, 4), np.int64), 10)
    check_tables(hip, 64, [], [], [], None, np.zeros((0, 0), np.int64), 0)
    check_tables(hip, 16, [5, 0, 16], [0, 0, 0], [], None, np.array([[3], [4], [5]]), 0)
    check_tables(hip, 16, [0, 0], [0, 0], [7], None, np.zeros((2, 0), np.int64), 4)


@pytest.mark.parametrize("requests", [5, 1500])
def test_tables_refuse_requests_alone(hip, requests):
    rng = np.random.default_rng(requests)
    cached, fresh, free, table = make_tables(rng, requests, 16, 100, 40, width=9)  # (some pass the table's width)
    cached[1], fresh[3] = -4, -2
    if requests > 1000:
        cached[1001], fresh[1002] = -1, -5
        fresh[700] = 2**31 - 1  # alone more rows than there are; their sum stops
        fresh[1200], cached[1300] = 2**31 - 1, 2**31 - 1
    rows = int(np.clip(fresh, 0, 100).sum())
    check_tables(hip, 16, cached, fresh, free, None, table, rows)
    check_tables(hip, 16, cached, fresh, free, None, table, rows // 2)      # too few rows
    check_tables(hip, 16, cached, fresh, free[:len(free) // 3], None, table, rows)  # too few pages
    check_tables(hip, 16, cached, fresh, free, len(free) - 4, table, rows)  # most of them taken before
    check_tables(hip, 16, cached, fresh, free, len(free) + 4, table, rows)
    check_tables(hip, 16, cached, fresh, free, -3, table, rows)
    odd = free.copy()
    odd[::3], odd[1::3] = -1, 2**31 - 7  # slots that cannot be
    check_tables(hip, 16, cached, fresh, odd, None, table, rows)


# ---- appending ------------------------------------------------------------------------------------------------------------------

class Pages:
    """A cache on the host and on the GPU, filled alike."""

    def __init__(self, hip, rng, pages, page, heads, dim, stale=None):
        self.hip, self.shape = hip, (pages, page, heads, dim)
        codes = lambda *shape: (plain.narrow(np.clip(rng.normal(size=shape) * 90, -448, 448)) if stale is None else np.full(shape, stale, np.uint8))
        self.k, self.v = codes(pages, heads, page, dim), codes(pages, heads, dim, page)
        self.k_scales, self.v_scales = (2.0 ** rng.integers(-9, -5, (pages, heads)).astype(np.float32) for _ in range(2))
        self.dev = [hip.DeviceBuffer.from_array(a) for a in (self.k, self.v, self.k_scales, self.v_scales)]
        self.cache = hip.KvCache(pages, page, heads, dim, *self.dev)

    def append(self, slots, k, v, kind, offset=0, extra=0, stream=None):
        """k, v: (rows, heads, dim) float32; rows of one matrix (k, then v, then `extra` values), beginning `offset` values in."""
        rows, width = len(slots), k.shape[1] * k.shape[2]
        both = np.concatenate([np.zeros((rows, offset)), k.reshape(rows, -1), v.reshape(rows, -1), np.zeros((rows, extra))], 1).astype(np.float32)
        raw = both if kind == "f32" else inputs.to_bf16(both)
        values = both if kind == "f32" else inputs.from_bf16(raw)
        buf, d_slots = self.hip.DeviceBuffer.from_array(raw), dev(self.hip, slots)
        call = self.hip.kv_cache_append_f32_dev if kind == "f32" else self.hip.kv_cache_append_bf16_dev
        call(self.cache, rows, d_slots, buf.at(offset * raw.itemsize), buf.at((offset + width) * raw.itemsize), raw.shape[1], stream=stream)
        self.hip.device_synchronize()
        plain.append(self.k, self.k_scales, slots, values[:, offset:offset + width].reshape(k.shape), False)
        plain.append(self.v, self.v_scales, slots, values[:, offset + width:offset + 2 * width].reshape(v.shape), True)

    def check(self, what=""):
        for name, buf, want in zip(("k", "v", "k_scales", "v_scales"), self.dev, (self.k, self.v, self.k_scales, self.v_scales)):
            got = buf.to_array(want.dtype, want.shape)
            if want.dtype == np.uint8:  # as values: one NaN is as good as another
                nan = (got & 127) == 127
                assert (nan == ((want & 127) == 127)).all(), f"{what}: {name}, NaN"
                same = nan | (got == want)
            else:
                same = got == want
            assert same.all(), f"{what}: {name} differs at {np.argwhere(~same)[:4].tolist()} ({(~same).sum()} values)"


def rows_for(rng, count, heads, dim):
    return [(rng.normal(size=(count, heads, dim)) * 2.0 ** rng.integers(-3, 4, (count, 1, 1))).astype(np.float32) for _ in range(2)]


APPENDS = [(4, 16, 1, 64), (5, 32, 3, 64), (6, 64, 2, 128), (3, 128, 2, 256), (4, 256, 1, 128), (9, 16, 5, 256)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("pages,page,heads,dim", APPENDS)
def test_append(hip, pages, page, heads, dim, kind):
    rng = np.random.default_rng(pages + page + dim)
    store = Pages(hip, rng, pages, page, heads, dim)
    order = rng.permutation(pages)
    p, o = int(order[0]), int(order[1])
    runs = {"one token": [p * page + 3], "a page anew": [p * page], "the next one": [p * page + 1], "a whole page": list(range(o * page, (o + 1) * page)),
            "the end of one and the beginning of the next": list(range(p * page + page - 5, (p + 1) * page)) + list(range(o * page, o * page + 7)),
            "one of each": [int(q) * page + int(rng.integers(0, page)) for q in order],
            "all pages": [int(q) * page + t for q in order for t in range(page)]}
    for what, slots in runs.items():
        store.append(slots, *rows_for(rng, len(slots), heads, dim), kind)
        store.check(what)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("pages,page,heads,dim", [(4, 16, 2, 64), (3, 64, 1, 128)])
def test_append_skips_repeats_and_any_order(hip, pages, page, heads, dim, kind):
    rng = np.random.default_rng(page)
    store = Pages(hip, rng, pages, page, heads, dim)
    for what, slots in {"none": [-1, -1], "outside": [pages * page, 2**31 - 1, -2**31, pages * page + 5], "between": [-1, 5, -1, page + 2, page + 3, -1],
                        "backwards": list(range(page - 1, -1, -1)), "twice": [2, 3, 2, 4, 3], "padding": [page + 1] + [2 * page] * 700,
                        "twice the first": [0, 5, 0], "shuffled": rng.permutation(page).tolist() + (page + rng.permutation(page)[:5]).tolist()}.items():
        store.append(slots, *rows_for(rng, len(slots), heads, dim), kind)
        store.check(what)


@pytest.mark.parametrize("kind,offset,extra", [("f32", 1, 0), ("f32", 4, 4), ("f32", 2, 1), ("bf16", 1, 0), ("bf16", 4, 0), ("bf16", 8, 8), ("bf16", 2, 3)])
def test_append_from_any_alignment(hip, kind, offset, extra):
    rng = np.random.default_rng(offset)
    store = Pages(hip, rng, 4, 32, 2, 64)
    slots = list(range(20, 75))
    store.append(slots, *rows_for(rng, len(slots), 2, 64), kind, offset, extra)
    store.check()


def test_scales_at_their_borders(hip):
    """Largest values on, just above and just below 448 times a power of two, tiny, huge and absent ones; a page that grows by steps."""
    rng = np.random.default_rng(3)
    store = Pages(hip, rng, 12, 16, 1, 64)
    above, below = np.nextafter(np.float32(448), np.float32(1e9)), np.nextafter(np.float32(448), np.float32(0))
    for i, largest in enumerate([448.0, above, below, 448.0 * 2.0**-20, float(above) * 2.0**-20, 0.0, 1e-45, 2.0**-118 * 449, 3e38, 1.0, 1.75]):
        for first in (0, 3):  # a page anew, and one that may grow
            k, v = (np.clip(x, -1, 1) * np.float32(min(1.0, largest)) for x in rows_for(rng, 2, 1, 64))
            k[1, 0, 7], v[0, 0, 9] = largest, -largest
            store.append([i * 16 + first, i * 16 + first + 1], k, v, "f32")
            store.check(f"{largest} at {first}")
    for step in range(40):  # every value doubles the scale now and then: what is held is rounded again
        k, v = (x * np.float32(1.37**step) for x in rows_for(rng, 1, 1, 64))
        store.append([11 * 16 + step % 16 if step else 11 * 16], k, v, "f32") if step % 16 else store.append([11 * 16], k, v, "f32")
        store.check(f"step {step}")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_values_that_are_not_numbers(hip, kind):
    rng = np.random.default_rng(5)
    store = Pages(hip, rng, 3, 16, 2, 64)
    k, v = rows_for(rng, 5, 2, 64)
    k[0, 0, 0], k[1, 1, 5], v[2, 0, 63], v[3, 1, 2], v[4, 1] = np.nan, np.inf, -np.inf, np.nan, np.nan
    store.append([16, 17, 18, 19, 36], k, v, kind)
    store.check("in a page anew and in another")
    k, v = rows_for(rng, 1, 2, 64)
    store.append([20], k * 100, v * 100, kind)
    store.check("NaN stays where a page grows")


# ---- attention ------------------------------------------------------------------------------------------------------------------

def check_attention(hip, rng, page, kv_heads, dim, group, lengths, fresh, causal, scale=None, behind=3, pages=None, width=None, edit=None,
                    stale=0x7f, extra=0, q_size=1.5, weight_step=2.0**-8, what=""):
    """A ragged batch over a cache whose places behind the lengths, and unused pages and their scales, hold NaN (`stale`)."""
    requests, heads = len(lengths), kv_heads * group
    used = [-(-max(0, n) // page) for n in lengths]
    width = max(used + [1]) if width is None else width
    pages = sum(used) + 2 if pages is None else pages
    store = Pages(hip, rng, pages, page, kv_heads, dim)
    order, at = np.append(1 + rng.permutation(pages - 1), 0), 0  # (page 0 stays unused: reads of pages that are none may go there)
    table = np.full((requests, width), SENTINEL)
    held = np.zeros((pages, page), bool)
    for r, n in enumerate(used):
        n = min(n, width)
        table[r, :n] = order[at:at + n]
        held[order[at:at + n]] = (np.arange(n * page) < lengths[r]).reshape(n, page)
        at += n
    if stale is not None:
        store.k[~held.any(1)], store.v[~held.any(1)] = stale, stale
        store.k_scales[~held.any(1)] = store.v_scales[~held.any(1)] = np.nan
        store.k.transpose(0, 2, 1, 3)[~held], store.v.transpose(0, 3, 1, 2)[~held] = stale, stale
    offsets = np.concatenate([[0], np.cumsum(fresh)])
    rows = int(offsets[-1]) + behind
    q_bits = inputs.to_bf16((q_size * rng.normal(size=(rows, heads * dim + 8 * extra))).astype(np.float32))
    if edit:
        edit(store, table, q_bits)
    for buf, array in zip(store.dev, (store.k, store.v, store.k_scales, store.v_scales)):
        buf.upload(array)
    ld_out = heads * dim + 4 * extra
    out = hip.DeviceBuffer.from_array(np.full((rows, ld_out), 0x4321, np.uint16))
    scale = 1.0 / np.sqrt(dim) if scale is None else scale
    d = [dev(hip, a) for a in (offsets, lengths, table)]
    d_q = hip.DeviceBuffer.from_array(q_bits)
    hip.attention_kv_cache_bf16_dev(store.cache, requests, rows, heads, scale, causal, *d, width, d_q, heads * dim + 8 * extra, out, ld_out)
    hip.device_synchronize()
    bits = out.to_array(np.uint16, (rows, ld_out))
    q = inputs.from_bf16(q_bits[:, :heads * dim].ravel()).astype(np.float64).reshape(rows, heads, dim)
    want, mine, bound = plain.attention(store.k, store.v, store.k_scales, store.v_scales, offsets, lengths, table, q, float(np.float32(scale)), causal,
                                        weight_step)
    assert (bits[~mine] == 0x4321).all() and (bits[:, heads * dim:] == 0x4321).all(), f"{what}: rows or columns behind the batch's"
    got = inputs.from_bf16(bits[:, :heads * dim].ravel()).astype(np.float64).reshape(rows, heads, dim)[mine]
    want, bound = want[mine], bound[mine]
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaN at {np.argwhere(np.isnan(got) != np.isnan(want))[:4].tolist()}"
    fine = ~np.isnan(want)
    err = np.abs(got - want)[fine]
    assert (err <= bound[fine]).all(), f"{what}: {(err > bound[fine]).sum()} of {err.size} outside, worst {np.max(err - bound[fine]):.3e}"
    return got


# page, kv_heads, dim, group, lengths, fresh rows
RAGGED = [
    (64, 1, 64, 1, [1], [1]), (64, 2, 128, 4, [1, 2, 63, 64, 65, 127, 128, 129], [1] * 8), (16, 3, 64, 2, [15, 16, 17, 31, 33, 100, 0, 5], [1] * 8),
    (32, 1, 256, 8, [200, 31, 32, 33], [1, 1, 1, 1]), (128, 2, 128, 1, [300, 5, 129], [1, 1, 1]), (256, 1, 64, 16, [1000, 256, 257], [1, 1, 1]),
    (64, 2, 64, 5, [70, 300, 20], [3, 17, 20]), (16, 1, 128, 3, [40, 40, 7], [40, 1, 7]), (32, 2, 256, 2, [90, 161], [33, 80]),
    (64, 1, 128, 32, [130, 77], [1, 2]), (64, 4, 64, 1, [500], [200]), (16, 1, 64, 7, [129, 0, 64, 1], [9, 0, 0, 1]),
    (64, 2, 128, 4, [640], [130]), (128, 1, 256, 1, [700, 140], [60, 130]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,kv_heads,dim,group,lengths,fresh", RAGGED)
def test_attention(hip, page, kv_heads, dim, group, lengths, fresh, causal):
    rng = np.random.default_rng(sum(lengths) + dim + group)
    check_attention(hip, rng, page, kv_heads, dim, group, lengths, fresh, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("requests", [63, 64, 65, 130, 4100])
def test_many_requests(hip, requests, causal):
    """Around the 64 requests, and 64 times 64, that one look at their offsets covers; some bring no row, some more than one."""
    rng = np.random.default_rng(requests)
    small = requests > 1000
    lengths, fresh = rng.integers(0, 9 if small else 90, requests), rng.integers(0, 3 if small else 5, requests)
    check_attention(hip, rng, 16, 1, 64, 2, lengths.tolist(), fresh.tolist(), causal)


@pytest.mark.parametrize("page,dim,kv_heads,group,length,fresh", [(64, 128, 1, 4, 5000, 1), (16, 64, 2, 1, 3001, 1), (256, 256, 1, 2, 2500, 2),
                                                                  (64, 64, 1, 8, 9000, 5), (32, 128, 2, 2, 1030, 20)])
def test_long_contexts(hip, page, dim, kv_heads, group, length, fresh):
    rng = np.random.default_rng(length)
    check_attention(hip, rng, page, kv_heads, dim, group, [length, 3, length // 2 + 1, 0], [fresh, 1, fresh, 1], True)
    # a table far wider than the batch needs
    check_attention(hip, rng, page, kv_heads, dim, group, [length // 3, 70], [fresh, 1], False, width=20000 // page)


@pytest.mark.parametrize("page,dim,kv_heads,group,lengths,fresh", [(64, 128, 1, 4, [2000, 130, 900, 0], [100, 70, 1, 40]), (16, 64, 2, 3, [1500, 64], [333, 50]),
                                                                   (128, 256, 1, 2, [1111, 2100], [200, 80]), (32, 128, 2, 1, [700, 1900], [700, 150]),
                                                                   (64, 64, 8, 1, [4096], [4096])])
def test_long_prompts(hip, page, dim, kv_heads, group, lengths, fresh):
    """Many rows of few requests, whose contexts are shared by several workgroups though rows have tiles of their own."""
    rng = np.random.default_rng(sum(lengths))
    for causal in (True, False) if max(fresh) < 1000 else (True,):
        check_attention(hip, rng, page, kv_heads, dim, group, lengths, fresh, causal)


@pytest.mark.parametrize("dim,kv_heads,group,fresh", [(128, 8, 4, 20), (64, 8, 8, 20), (256, 7, 4, 18)])
def test_many_prompts_of_uneven_lengths(hip, dim, kv_heads, group, fresh):
    """More wide tiles than the chip holds at once, two contexts of which are long enough to be cut."""
    rng = np.random.default_rng(dim)
    lengths = [int(n) for n in rng.integers(0, 90, 64)]
    lengths[7], lengths[40] = 3000, 2111
    for causal in (True, False):
        check_attention(hip, rng, 64, kv_heads, dim, group, lengths, [fresh] * 64, causal)


@pytest.mark.parametrize("requests,dim,kv_heads,group", [(65, 64, 2, 1), (130, 128, 1, 4), (600, 64, 1, 2), (70, 256, 1, 2)])
def test_many_requests_of_long_contexts(hip, requests, dim, kv_heads, group):
    """More than 64 requests, with contexts long enough that some are cut; some bring no row, some several."""
    rng = np.random.default_rng(requests + dim)
    lengths, fresh = rng.integers(300, 1000, requests), rng.integers(0, 3, requests)
    lengths[rng.permutation(requests)[:4]] = 5000, 4095, 3001, 4500
    for causal in (True, False):
        check_attention(hip, rng, 64, kv_heads, dim, group, lengths.tolist(), fresh.tolist(), causal)


@pytest.mark.parametrize("requests,dim", [(1100, 64), (700, 128)])
def test_a_long_context_among_very_many(hip, requests, dim):
    """The one long context is first, last and between, and short ones are next to it."""
    rng = np.random.default_rng(requests)
    for at in (0, requests // 2 + 1, requests - 1):
        lengths = rng.integers(0, 20, requests)
        lengths[at] = 9000
        check_attention(hip, rng, 16, 6, dim, 1, lengths.tolist(), [1] * requests, True)


@pytest.mark.parametrize("dim,group,length,fresh", [(64, 1, 32700, 1), (128, 1, 65530, 2), (256, 1, 32768, 1), (64, 16, 40000, 1), (128, 16, 32701, 1),
                                                    (64, 4, 12200, 70), (128, 4, 12280, 70), (256, 4, 12200, 35), (128, 2, 20000, 40)])
def test_as_many_parts_as_there_can_be(hip, dim, group, length, fresh):
    """One context on one key head, cut into up to 128 parts of narrow tiles of columns or up to 16 of wide ones, whose shares then grow."""
    check_attention(hip, np.random.default_rng(length), 256, 1, dim, group, [length], [fresh], True)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_prompts_among_many_requests(hip, dim):
    """More than 64 requests, three of them with prompts that are cut, beside single tokens and requests that wait."""
    rng = np.random.default_rng(dim)
    lengths, fresh = rng.integers(1, 200, 90), rng.integers(0, 2, 90)
    for r, n, rows in ((3, 2500, 75), (64, 1800, 80), (89, 3000, 70)):
        lengths[r], fresh[r] = n, rows
    check_attention(hip, rng, 64, 1, dim, 2, lengths.tolist(), fresh.tolist(), True)


@pytest.mark.parametrize("kv_heads,dim,length", [(520, 64, 700), (400, 64, 1500), (200, 128, 900), (260, 256, 400)])
def test_many_key_heads(hip, kv_heads, dim, length):
    """As many key heads as there should be workgroups, and more and fewer."""
    check_attention(hip, np.random.default_rng(kv_heads), 64, kv_heads, dim, 1, [length, 20], [1, 2], True)


def test_rows_without_keys(hip):
    """More rows than tokens: the first see none, and are 0; requests of no length, of a negative one."""
    rng = np.random.default_rng(1)
    for dim in (64, 128, 256):
        got = check_attention(hip, rng, 16, 2, dim, 3, [5, 0, -3, 20], [30, 4, 2, 45], True)
        assert (got[:25] == 0).all() and (got[30:36] == 0).all() and (got[26:30] != 0).any()
        check_attention(hip, rng, 16, 2, dim, 3, [0, 0, -2**31], [3, 1, 1], False)


@pytest.mark.parametrize("requests,rows,dim,group", [(8, 40, 64, 1), (130, 50, 64, 2), (6, 300, 64, 1), (200, 700, 128, 1), (7, 130, 256, 2)])
def test_row_offsets_out_of_order(hip, requests, rows, dim, group):
    """Offsets that rise and fall claim more tiles of columns than the rows have: nothing behind the rows is written, and the calls after it, which
    count in the same places, are right."""
    rng = np.random.default_rng(rows)
    store = Pages(hip, rng, 20, 64, 1, dim)
    width = 40
    d_q = hip.DeviceBuffer.from_array(inputs.to_bf16(rng.normal(size=(rows, group * dim)).astype(np.float32)))
    out = hip.DeviceBuffer.from_array(np.full((rows + 9, group * dim), 0x4321, np.uint16))
    d_table, d_lengths = dev(hip, rng.integers(0, 20, (requests, width))), dev(hip, rng.integers(1000, 2500, requests))
    offsets = np.where(np.arange(requests + 1) % 2 == 1, rows, 0)
    for causal in (True, False):
        hip.attention_kv_cache_bf16_dev(store.cache, requests, rows, group, 0.1, causal, dev(hip, offsets), d_lengths, d_table, width, d_q, group * dim,
                                        out, group * dim)
        hip.device_synchronize()
        assert (out.to_array(np.uint16, (rows + 9, group * dim))[rows:] == 0x4321).all()
        check_attention(hip, rng, 64, 1, dim, group, [2100, 5, 1500], [1, 1, 2], causal)
        check_attention(hip, rng, 64, 1, dim, group, [1500, 300], [rows // 2, 1], causal)


def test_lengths_beyond_the_table(hip):
    rng = np.random.default_rng(2)
    for causal in (True, False):
        # the table's two pages are what counts; 2^31 - 1 tokens are not reached for
        store_pages = 6
        check_attention(hip, rng, 64, 1, 64, 2, [128, 64], [2, 2], causal, pages=store_pages, width=2,
                        edit=lambda store, table, q: table.__setitem__((1, 1), 5))
    lengths = [2**31 - 1, 500]
    rng = np.random.default_rng(3)
    store = Pages(hip, rng, 4, 64, 1, 64)
    table = np.array([[2, 0], [3, 1]])
    q_bits = inputs.to_bf16(rng.normal(size=(4, 64)).astype(np.float32))
    out = hip.DeviceBuffer.from_array(np.zeros((4, 64), np.uint16))
    hip.attention_kv_cache_bf16_dev(store.cache, 2, 4, 1, 0.125, False, dev(hip, [0, 2, 4]), dev(hip, lengths), dev(hip, table), 2,
                                    hip.DeviceBuffer.from_array(q_bits), 64, out, 64)
    hip.device_synchronize()
    q = inputs.from_bf16(q_bits.ravel()).astype(np.float64).reshape(4, 1, 64)
    want, _, bound = plain.attention(store.k, store.v, store.k_scales, store.v_scales, [0, 2, 4], lengths, table, q, 0.125, False)
    assert (np.abs(inputs.from_bf16(out.to_array(np.uint16, (4, 64)).ravel()).reshape(4, 1, 64) - want) <= bound).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_pages_outside_the_cache(hip, dim, causal):
    """Their tokens are left out, whatever the entry says; a request all of whose pages are outside sees nothing."""
    rng = np.random.default_rng(4)

    def edit(store, table, q):
        table[0, 1], table[0, 3], table[1, 0] = -1, 2**31 - 1, -2**31
        table[2, :] = len(store.k)

    got = check_attention(hip, rng, 32, 2, dim, 2, [150, 40, 60], [4, 20, 3], causal, edit=edit)
    assert (got[24:] == 0).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_numbers_that_are_none(hip, dim):
    """NaN in a key reaches the rows that see the key, in a value its column of them, in a query its head; nothing else.  A key's NaN hidden by
    the mask, in the tile the diagonal runs through, reaches nobody."""
    rng = np.random.default_rng(6)

    def edit(store, table, q):
        store.v[table[0, 3], 0, 5, 40 % 16] = 0x7f      # token 3 * 16 + 8 of request 0
        store.v[table[0, 5], 1, 2, 4] = 0xff            # token 84
        store.k[table[0, 5], 1, 9, 1] = 0x7f            # token 89
        q[60, 3] = 0x7fc0

    got = check_attention(hip, rng, 16, 2, dim, 2, [100, 90], [40, 40], True, edit=edit, stale=0x7f)
    assert np.isnan(got).any() and not np.isnan(got).all()
    check_attention(hip, rng, 16, 2, dim, 2, [100, 90], [40, 40], False, edit=edit, stale=0xff)


@pytest.mark.parametrize("dim,group,lengths,fresh", [(64, 4, [700, 90], [1, 3]), (128, 4, [6000, 5], [1, 1]), (256, 2, [900, 2000], [2, 10]), (64, 16, [500], [8])])
def test_weights_of_few_rows(hip, dim, group, lengths, fresh):
    """Two pieces of bf16 hold a weight: the first is off by 2^-8 of it at the most, the second by 2^-8 of that."""
    check_attention(hip, np.random.default_rng(dim), 64, 2, dim, group, lengths, fresh, True, weight_step=2.0**-16)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-30])
def test_scales_of_the_scores(hip, scale):
    rng = np.random.default_rng(7)
    for causal in (True, False):
        check_attention(hip, rng, 64, 1, 128, 4, [200, 17], [5, 17], causal, scale=scale)


@pytest.mark.parametrize("scale", [0.0, 1e-45, 1e-41, -1e-38, 1e-36])
def test_small_scales_of_large_scores(hip, scale):
    """Products of queries and keys of 10^36, on narrow tiles of columns and on wide ones, with masked keys beside them."""
    def edit(store, table, q):
        store.k_scales[table[table >= 0]] = 2.0**60

    rng = np.random.default_rng(24)
    for dim in (64, 128, 256):
        for lengths, fresh in (([200, 17], [5, 17]), ([300], [150])):
            check_attention(hip, rng, 64, 1, dim, 2, lengths, fresh, True, scale=scale, edit=edit, q_size=1e15)


def test_strides(hip):
    rng = np.random.default_rng(8)
    for extra in (1, 3):
        check_attention(hip, rng, 64, 2, 64, 3, [100, 64, 9], [1, 20, 2], True, extra=extra, behind=9)


def test_pages_of_very_different_sizes(hip):
    """Scales of 2^-100 and 2^40 beside each other, and the largest and smallest there are."""
    rng = np.random.default_rng(9)

    def edit(store, table, q):
        store.v_scales[table[0, ::2]], store.v_scales[table[0, 1::2]] = 2.0**-100, 2.0**40
        store.k_scales[table[1, :6:2]] = 2.0**-118
        store.v_scales[table[1, :6]] = 2.0**110

    check_attention(hip, rng, 16, 2, 64, 2, [100, 90], [3, 50], True, edit=edit)


@pytest.mark.parametrize("dim,kv_heads,group,lengths,fresh", [(64, 2, 2, [300, 7], [1, 3]), (128, 1, 4, [5000, 900], [1, 2]), (256, 1, 2, [2500, 40], [2, 1]),
                                                              (64, 1, 8, [400, 30], [60, 2]), (128, 2, 4, [2600, 500], [40, 33]), (256, 1, 4, [1500], [70])])
def test_averages_of_values_near_the_largest(hip, dim, kv_heads, group, lengths, fresh):
    """Their sum is beyond f32, their average is not: on all pages, on the later ones alone, and on every fourth beside pages of 2^-20."""
    def edit(where):
        def change(store, table, q):
            store.v[...] &= 0x7f
            for r, n in enumerate(lengths):
                pages = table[r, :-(-n // 64)]
                store.v_scales[pages] = 2.0**-20
                store.v_scales[pages[where(len(pages))]] = 2.0**119
        return change

    for where in (lambda n: slice(None), lambda n: slice(n // 2, None), lambda n: slice(n % 4, None, 4)):
        got = check_attention(hip, np.random.default_rng(23), 64, kv_heads, dim, group, lengths, fresh, True, edit=edit(where))
        assert np.isfinite(got).all() and got.max() > 2.0**120


def test_a_page_beyond_32_bits(hip):
    """Codes more than 2^32 bytes into the cache's memory, appended and read."""
    pages, page, heads, dim = 2200, 256, 32, 256  # 4.6 GB each of keys and values
    store = hip.KvCache(pages, page, heads, dim)
    rng = np.random.default_rng(10)
    last = pages - 1
    host_k, host_v = np.zeros((1, heads, page, dim), np.uint8), np.zeros((1, heads, dim, page), np.uint8)
    scales = [np.zeros((1, heads), np.float32) for _ in range(2)]
    rows = rows_for(rng, 100, heads, dim)
    raw = [inputs.to_bf16(x.reshape(100, -1)) for x in rows]
    values = [inputs.from_bf16(r.ravel()).reshape(100, heads, dim) for r in raw]
    slots = last * page + np.arange(100)
    d_k, d_v = (hip.DeviceBuffer.from_array(r) for r in raw)
    hip.kv_cache_append_bf16_dev(store, 100, dev(hip, slots), d_k, d_v, heads * dim)
    plain.append(host_k, scales[0], np.arange(100), values[0], False)
    plain.append(host_v, scales[1], np.arange(100), values[1], True)
    for n in (2, 100):  # a narrow tile of columns, and a wide one
        q_bits = inputs.to_bf16(rng.normal(size=(n, heads * dim)).astype(np.float32))
        out = hip.DeviceBuffer(n * heads * dim * 2)
        hip.attention_kv_cache_bf16_dev(store, 1, n, heads, 1 / 16, True, dev(hip, [0, n]), dev(hip, [100]), dev(hip, [[last]]), 1,
                                        hip.DeviceBuffer.from_array(q_bits), heads * dim, out, heads * dim)
        hip.device_synchronize()
        q = inputs.from_bf16(q_bits.ravel()).astype(np.float64).reshape(n, heads, dim)
        want, _, bound = plain.attention(host_k, host_v, *scales, [0, n], [100], np.array([[0]]), q, 1 / 16, True)
        got = inputs.from_bf16(out.to_array(np.uint16, n * heads * dim)).reshape(n, heads, dim)
        assert (np.abs(got - want) <= bound).all(), n


# ---- a run of them together -------------------------------------------------------------------------------------------------------

class Server:
    """A model's attention as it would be served: tables, rotary positions in place in the fused projection, append, attention."""

    def __init__(self, hip, rng, requests, rows, page=16, kv_heads=2, group=3, dim=64, pages=60, width=12):
        self.hip, self.rng, self.requests, self.rows, self.page, self.width = hip, rng, requests, rows, page, width
        self.kv_heads, self.heads, self.dim = kv_heads, kv_heads * group, dim
        self.store = Pages(hip, rng, pages, page, kv_heads, dim, stale=0x7f)
        self.free = rng.permutation(pages)
        self.config = {"rotary_dim": dim, "base": 10000.0}
        self.rotary = hip.Rotary(**self.config)
        self.ld = (self.heads + 2 * kv_heads) * dim
        buf = lambda n: dev(hip, np.full(n, SENTINEL))
        self.d_cached, self.d_fresh, self.d_free, self.d_table = buf(requests), buf(requests), dev(hip, self.free), buf(requests * width)
        self.d_offsets, self.d_lengths, self.d_positions, self.d_slots, self.d_counts = buf(requests + 1), buf(requests), buf(rows), buf(rows), buf(3)
        self.d_taken = dev(hip, [0])
        self.d_qkv, self.d_out = hip.DeviceBuffer(rows * self.ld * 2), hip.DeviceBuffer(rows * self.heads * dim * 2)
        self.cached, self.taken, self.table = np.zeros(requests, np.int64), 0, np.full((requests, width), SENTINEL)

    def feed(self, fresh):
        self.fresh = np.asarray(fresh)
        self.qkv = inputs.to_bf16(self.rng.normal(size=(self.rows, self.ld)).astype(np.float32))
        self.d_cached.upload(self.cached.astype(np.int32))
        self.d_fresh.upload(self.fresh.astype(np.int32))
        self.d_taken.upload(np.array([self.taken], np.int32))
        self.d_qkv.upload(self.qkv)

    def step(self, stream=None):
        hip, d = self.hip, self.dim
        hip.page_tables_dev(self.requests, self.page, self.d_cached, self.d_fresh, len(self.free), self.d_free, self.d_taken, self.width, self.d_table,
                            self.rows, self.d_offsets, self.d_lengths, self.d_positions, self.d_slots, self.d_counts, stream=stream)
        hip.rotary_bf16_dev(self.rows, self.heads + self.kv_heads, d, self.rotary, self.d_positions, self.d_qkv, self.ld, self.d_qkv, self.ld, stream=stream)
        k, v = (self.d_qkv.at((self.heads + i * self.kv_heads) * d * 2) for i in (0, 1))
        hip.kv_cache_append_bf16_dev(self.store.cache, self.rows, self.d_slots, k, v, self.ld, stream=stream)
        hip.attention_kv_cache_bf16_dev(self.store.cache, self.requests, self.rows, self.heads, d**-0.5, True, self.d_offsets, self.d_lengths,
                                        self.d_table, self.width, self.d_qkv, self.ld, self.d_out, self.heads * d, stream=stream)

    def check(self, what):
        """What the step should have done, from the queries and keys that the GPU turned (whose own test is above: their rounding to
        bf16 would otherwise meet another's a step away)."""
        offsets, lengths, positions, slots, counts, self.table = plain.page_tables(self.page, self.cached, self.fresh, self.free, self.taken, self.table,
                                                                                     self.rows)
        used = counts[1]
        assert self.d_lengths.to_array(np.int32, self.requests).tolist() == lengths, what
        assert self.d_slots.to_array(np.int32, self.rows).tolist()[:used] == slots[:used], what
        d, n = self.dim, self.heads + self.kv_heads
        after = inputs.from_bf16(self.d_qkv.to_array(np.uint16, (self.rows, self.ld)).ravel()).astype(np.float64).reshape(self.rows, -1, d)
        before = inputs.from_bf16(self.qkv.ravel()).astype(np.float64).reshape(self.rows, -1, d)
        want, size = plain.rotary(before[:used, :n], positions[:used], d, False, plain.turns(d))
        assert (np.abs(after[:used, :n] - want) <= 8 * 2.0**-24 * size + 2.0**-8 * np.abs(want)).all(), what
        assert (after[:, n:] == before[:, n:]).all(), what
        for codes, scales, first, transposed in ((self.store.k, self.store.k_scales, self.heads, False), (self.store.v, self.store.v_scales, n, True)):
            plain.append(codes, scales, slots[:used], after[:used, first:first + self.kv_heads], transposed)
        self.store.check(what)
        want, mine, bound = plain.attention(self.store.k, self.store.v, self.store.k_scales, self.store.v_scales, offsets, lengths, self.table,
                                            after[:, :self.heads], float(np.float32(d**-0.5)), True)
        got = inputs.from_bf16(self.d_out.to_array(np.uint16, self.rows * self.heads * d)).reshape(self.rows, self.heads, d)
        assert (np.abs(got[mine] - want[mine]) <= bound[mine]).all(), what
        self.cached, self.taken = np.asarray(lengths), counts[0]


STEPS = [[20, 1, 0, 33], [1, 16, 5, 1], [1, 1, 1, 1], [1, 0, 1, 20], [1, 1, 1, 1]]


def test_serving(hip):
    server = Server(hip, np.random.default_rng(11), 4, 60)
    for i, fresh in enumerate(STEPS):
        server.feed(fresh)
        server.step()
        hip.device_synchronize()
        server.check(f"step {i}")


def test_serving_on_a_stream(hip):
    server = Server(hip, np.random.default_rng(12), 4, 60, page=32, dim=128, kv_heads=1, group=4)
    stream = hip.Stream()
    for i, fresh in enumerate(STEPS):
        server.feed(fresh)
        server.step(stream)
        stream.synchronize()
        server.check(f"step {i}")
    hip.release_scratch(stream)


def test_serving_from_a_graph(hip):
    """One recorded step replayed over growing contexts, with eager calls on other data between the replays."""
    import torch
    server, other = (Server(hip, np.random.default_rng(seed), 4, 60, pages=400, width=100) for seed in (13, 14))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        server.step(torch.cuda.current_stream().cuda_stream)
    try:
        for i, fresh in enumerate(STEPS + [[1, 1, 1, 1]] * 3):
            server.feed(fresh)
            other.feed(fresh)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            other.step()
            torch.cuda.synchronize()
            server.check(f"replay {i}")
            other.check(f"eager {i}")
    finally:
        del graph
        hip.release_scratch(stream.cuda_stream)
        hip.release_scratch(None)


@pytest.mark.parametrize("rows", [1, 90])
def test_contexts_of_a_graph(hip, rows):
    """Two recorded calls of one stream, of different sizes, replayed in turn over contexts that one workgroup takes and that several share,
    with eager calls between."""
    import torch
    rng = np.random.default_rng(rows)
    dim, kv_heads, group, page = 64, 2, 2, 64
    heads, width = kv_heads * group, 40
    store = Pages(hip, rng, 100, page, kv_heads, dim)
    requests = [3, 2]
    tables = [rng.permutation(100)[:r * width].reshape(r, width) for r in (2, 2)]
    tables = [np.concatenate([tables[0], tables[0][:1]]), tables[1]]
    offsets = [np.arange(r + 1) * rows for r in requests]
    q_bits = [inputs.to_bf16(rng.normal(size=(r * rows, heads * dim)).astype(np.float32)) for r in requests]
    d_offsets, d_tables, d_q = ([dev(hip, a) for a in offsets], [dev(hip, a) for a in tables], [hip.DeviceBuffer.from_array(a) for a in q_bits])
    d_lengths = [dev(hip, np.zeros(r)) for r in requests]
    outs = [hip.DeviceBuffer(r * rows * heads * dim * 2) for r in requests]

    def call(i, stream=None):
        hip.attention_kv_cache_bf16_dev(store.cache, requests[i], requests[i] * rows, heads, 0.125, True, d_offsets[i], d_lengths[i], d_tables[i], width,
                                        d_q[i], heads * dim, outs[i], heads * dim, stream=stream)

    def check(i, lengths, what):
        want, mine, bound = plain.attention(store.k, store.v, store.k_scales, store.v_scales, offsets[i], lengths, tables[i],
                                            inputs.from_bf16(q_bits[i].ravel()).astype(np.float64).reshape(-1, heads, dim), 0.125, True)
        got = inputs.from_bf16(outs[i].to_array(np.uint16, requests[i] * rows * heads * dim)).reshape(-1, heads, dim)
        assert mine.all() and (np.abs(got - want) <= bound).all(), what

    graphs, stream = [torch.cuda.CUDAGraph() for _ in requests], torch.cuda.Stream()
    torch.cuda.synchronize()
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, stream=stream):
            call(i, torch.cuda.current_stream().cuda_stream)
    try:
        for lengths in ([2560, 700, 3], [1, 0, 2], [64, 2560, 2500], [2000, 2000, 2000]):
            for i, r in enumerate(requests):
                d_lengths[i].upload(np.array(lengths[:r], np.int32))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for graph in graphs * 2:
                    graph.replay()
            torch.cuda.synchronize()
            for i, r in enumerate(requests):
                check(i, lengths[:r], f"replay of {i}, {lengths}")
                call(i)
                hip.device_synchronize()
                check(i, lengths[:r], f"eager {i}, {lengths}")
    finally:
        del graphs, graph
        hip.release_scratch(stream.cuda_stream)
        hip.release_scratch(None)


def test_two_streams_from_two_threads(hip):
    """Steps on two streams at once, each from a thread of its own, with contexts that several workgroups share: nothing of theirs meets."""
    import threading
    rng = np.random.default_rng(21)
    dim, kv_heads, group, page, width = 128, 2, 4, 64, 60
    heads = kv_heads * group
    store = Pages(hip, rng, 150, page, kv_heads, dim)
    works, errors = [], []
    for rows, lengths in ((1, [3800, 100, 2000]), (40, [3000, 2500])):
        n = len(lengths)
        table = rng.integers(0, 150, (n, width))
        q_bits = inputs.to_bf16(rng.normal(size=(n * rows, heads * dim)).astype(np.float32))
        q = inputs.from_bf16(q_bits.ravel()).astype(np.float64).reshape(-1, heads, dim)
        offsets = np.arange(n + 1) * rows
        want = plain.attention(store.k, store.v, store.k_scales, store.v_scales, offsets, lengths, table, q, 0.09, True)
        works.append((n, rows, hip.Stream(), [dev(hip, a) for a in (offsets, lengths, table)], hip.DeviceBuffer.from_array(q_bits),
                      hip.DeviceBuffer(q_bits.nbytes), want))

    def serve(n, rows, stream, d, d_q, out, want):
        try:
            for i in range(30):
                hip.attention_kv_cache_bf16_dev(store.cache, n, n * rows, heads, 0.09, True, *d, width, d_q, heads * dim, out, heads * dim, stream=stream)
                if i % 10 == 9:
                    stream.synchronize()
                    got = inputs.from_bf16(out.to_array(np.uint16, n * rows * heads * dim)).reshape(-1, heads, dim)
                    assert (np.abs(got - want[0]) <= want[2]).all(), (rows, i)
            hip.release_scratch(stream)
        except BaseException as e:
            errors.append(e)

    hip.device_synchronize()
    threads = [threading.Thread(target=serve, args=w) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_the_same_twice(hip):
    """Whichever workgroup puts a context's parts together, the bits are the same."""
    rng = np.random.default_rng(22)
    for rows, dim, page in ((1, 128, 64), (3, 256, 16), (80, 64, 32)):
        lengths = [int(n) for n in rng.integers(600, 4000, 3)]
        seeds = [check_attention(hip, np.random.default_rng(5), page, 2, dim, 2, lengths, [rows] * 3, True) for _ in range(4)]
        assert all((s == seeds[0]).all() for s in seeds)
