"""Calls around the paged 8-bit cache that are refused before anything is launched: the library's host code on a runtime that runs
nothing (runtime_stub.cpp), so that no GPU is needed."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

PRELUDE = """
import ctypes, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
from spiraltorch_amd import _lib, hip
launches = ctypes.c_ulonglong.in_dll(stub, "stub_launches")
no_memory = ctypes.c_int.in_dll(stub, "stub_no_memory")
grid = ctypes.c_uint.in_dll(stub, "stub_grid")
M = 1 << 20
def cache(pages=8, page=64, heads=2, dim=64, k=16 * M, v=32 * M, ks=48 * M, vs=64 * M):
    return hip.KvCache(pages, page, heads, dim, k, v, ks, vs)
def refused(call, *args, **kw):
    before = launches.value
    try:
        call(*args, **kw)
    except hip.HipErr as e:
        assert launches.value == before, "launched"
        return {2: "invalid", 4: "nonfinite", 5: "unsupported"}[e.status]
    return "taken"
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("stub") / "libstub.so")
    subprocess.run(["hipcc", "-shared", "-fPIC", "-O1", "-x", "hip", "--offload-host-only", os.path.join(ROOT, "tests", "runtime_stub.cpp"), "-o", path], check=True)
    return path


def run(stub, body):
    done = subprocess.run([sys.executable, "-c", PRELUDE + body, stub], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout.split()


def answers(stub, call, base, changes):
    """What `call` says to the arguments of `base` with each of `changes` made to them."""
    return run(stub, f"""
base = dict({base})
for change in ({', '.join(f'dict({c})' for c in changes)},):
    print(refused({call}, **{{**base, **change}}))
""")


def test_page_tables(stub):
    base = ("requests=4, page_size=64, cached=1*M, fresh=2*M, free_count=10, free_pages=3*M, taken_before=4*M, table_width=8, page_table=5*M, rows=16, "
            "row_offsets=6*M, lengths=7*M, positions=8*M, slots=9*M, counts=10*M")
    expected = {"": "taken", "requests=0": "taken", "rows=0, positions=None, slots=None": "taken", "free_count=0, free_pages=None": "taken",
                "taken_before=None": "taken", "table_width=0, page_table=None": "taken",
                "requests=0, cached=None, fresh=None, lengths=None, page_table=None": "taken",
                "page_size=0": "unsupported", "page_size=8": "unsupported", "page_size=48": "unsupported", "page_size=512": "unsupported",
                "requests=2**31": "unsupported", "rows=2**31": "unsupported", "free_count=2**31": "unsupported", "table_width=2**31": "unsupported",
                "requests=2**40, table_width=2**40": "invalid",
                "cached=None": "invalid", "fresh=None": "invalid", "lengths=None": "invalid", "counts=None": "invalid", "row_offsets=None": "invalid",
                "positions=None": "invalid", "slots=None": "invalid", "page_table=None": "invalid", "free_pages=None": "invalid",
                "lengths=1*M": "invalid", "counts=4*M": "invalid", "counts=4*M - 8": "invalid", "counts=4*M + 4": "taken", "counts=4*M - 12": "taken",
                "positions=9*M": "invalid", "slots=8*M + 60": "invalid", "slots=8*M + 64": "taken", "page_table=3*M - 124": "invalid",
                "page_table=3*M - 128": "taken"}
    assert answers(stub, "hip.page_tables_dev", base, expected) == list(expected.values())


def test_rotary(stub):
    for call, size in (("hip.rotary_f32_dev", 4), ("hip.rotary_bf16_dev", 2)):
        base = "rows=3, heads=2, head_dim=64, rotary=hip.Rotary(64), positions=1*M, src=2*M, ld_in=128, dst=3*M, ld_out=128"
        expected = {"": "taken", "rotary=hip.Rotary(0)": "taken", "rotary=hip.Rotary(62)": "taken", "dst=2*M": "taken", "ld_in=200, ld_out=333": "taken",
                    "positions=None, sequence=5": "taken", "positions=None": "invalid", "rows=0, src=None, dst=None, positions=None": "taken",
                    "rotary=hip.Rotary(63)": "invalid", "rotary=hip.Rotary(66)": "invalid", "rotary=hip.Rotary(64, base=0.5)": "invalid",
                    "rotary=hip.Rotary(64, base=float('nan'))": "invalid", "rotary=hip.Rotary(64, factor=0.0)": "invalid",
                    "rotary=hip.Rotary(64, factor=float('inf'))": "invalid", "rotary=hip.Rotary(64, magnitude=float('inf'))": "invalid",
                    "rotary=hip.Rotary(64, original_length=-1.0)": "invalid",
                    "rotary=hip.Rotary(64, original_length=9.0, low_turns=4.0, high_turns=4.0)": "invalid",
                    "rotary=hip.Rotary(64, original_length=0.0, low_turns=4.0, high_turns=4.0)": "taken",
                    "src=None": "invalid", "dst=None": "invalid", "ld_in=127": "invalid", "ld_out=127": "invalid",
                    "head_dim=1026, ld_in=4096, ld_out=4096": "unsupported", "rows=2**40": "unsupported", "rows=2**62": "invalid",
                    "rows=2**31 - 1, ld_in=2**31 - 1": "invalid", "rows=2**31 - 1, ld_out=2**31 - 1": "invalid",
                    # overlaps: other strides, shifted, columns that meet and that do not
                    "dst=2*M, ld_out=256": "invalid", f"dst=2*M + {size}": "invalid",
                    f"ld_in=256, ld_out=256, dst=2*M + {128 * size}": "taken", f"ld_in=256, ld_out=256, dst=2*M + {127 * size}": "invalid",
                    f"ld_in=256, ld_out=256, dst=2*M - {128 * size}": "taken", f"ld_in=256, ld_out=256, dst=2*M + {129 * size}": "invalid",
                    f"ld_in=300, ld_out=300, dst=2*M + {300 * size}": "invalid", f"ld_in=300, ld_out=300, dst=2*M + {450 * size}": "taken"}
        assert answers(stub, call, base, expected) == list(expected.values())


CACHES = {"cache=cache(page=8)": "unsupported", "cache=cache(page=96)": "unsupported", "cache=cache(dim=32)": "unsupported", "cache=cache(dim=96)": "unsupported",
          "cache=cache(k=8 + M)": "unsupported", "cache=cache(v=4 + M)": "unsupported", "cache=cache(k=0)": "invalid", "cache=cache(vs=0)": "invalid",
          "cache=cache(pages=2**31)": "unsupported", "cache=cache(heads=2**32)": "unsupported",
          "cache=cache(pages=2**20, heads=2**12)": "unsupported"}


def test_append(stub):
    for call in ("hip.kv_cache_append_f32_dev", "hip.kv_cache_append_bf16_dev"):
        base = "cache=cache(), rows=5, slots=1*M, k=2*M, v=3*M, ld=128"
        expected = {"": "taken", "ld=131, k=2*M + 2": "taken", "rows=0, slots=None, k=None, v=None": "taken", "slots=None": "invalid", "k=None": "invalid",
                    "v=None": "invalid", "ld=127": "invalid", "rows=2**31": "unsupported", "ld=2**40": "unsupported", "rows=2**40, ld=2**40": "invalid", "rows=2**31 - 300, ld=2**31 - 1": "invalid",
                    # rows within the cache's 65536 bytes of keys or values, or its 64 of scales
                    "k=16*M + 65532": "invalid", "k=16*M + 65536": "taken", "v=32*M": "invalid", "k=48*M - 8": "invalid", "v=64*M + 60": "invalid",
                    "v=64*M + 64": "taken", **CACHES}
        assert answers(stub, call, base, expected) == list(expected.values())


def test_append_of_the_most_rows(stub):
    """The kernel's row numbers go up to 512 beyond the rows, within int32."""
    for call in ("hip.kv_cache_append_f32_dev", "hip.kv_cache_append_bf16_dev"):
        base = "cache=cache(page=256, dim=256), rows=5, slots=2**44, k=2**46, v=2**47, ld=512"
        expected = {"rows=2**31 - 1 - 512": "taken", "rows=2**31 - 512": "unsupported", "rows=2**31 - 1 - 256": "unsupported"}
        assert answers(stub, call, base, expected) == list(expected.values())


def test_attention(stub):
    base = ("cache=cache(), requests=3, rows=7, heads=4, scale=0.1, causal=True, row_offsets=1*M, lengths=2*M, page_table=3*M, table_width=4, "
            "q=4*M, ld_q=256, out=5*M, ld_out=256")
    expected = {"": "taken", "causal=False": "taken", "heads=2, ld_q=128, ld_out=132": "taken", "rows=0, q=None, out=None": "taken",
                "requests=0": "taken", "table_width=0, page_table=None": "taken", "scale=-1.0": "taken", "scale=0.0": "taken",
                "heads=0": "invalid", "heads=3": "invalid", "heads=1": "invalid", "scale=float('nan')": "nonfinite", "scale=float('inf')": "nonfinite",
                "row_offsets=None": "invalid", "lengths=None": "invalid", "page_table=None": "invalid", "q=None": "invalid", "out=None": "invalid",
                "ld_q=255": "invalid", "ld_q=248": "invalid", "ld_out=252": "invalid", "ld_q=257": "unsupported", "ld_out=258": "unsupported",
                "q=4*M + 8": "unsupported", "out=5*M + 4": "unsupported", "out=5*M + 8": "taken",
                "rows=2**30": "unsupported", "rows=2**63": "invalid", "requests=2**31": "unsupported", "requests=2**62": "invalid",
                "out=4*M": "invalid", "out=4*M + 512": "invalid", "ld_q=512, ld_out=512, out=4*M + 512": "taken",
                "rows=2**29 - 1, heads=4, ld_q=2**31 - 8, ld_out=2**31 - 4": "invalid", "out=16*M + 65528": "invalid", "out=16*M + 65536": "taken",
                "out=32*M - 8": "invalid", "out=64*M": "invalid", **CACHES}
    assert answers(stub, "hip.attention_kv_cache_bf16_dev", base, expected) == list(expected.values())


def test_attention_scales(stub):
    """A scale that f32 holds, but not times log2(e)."""
    base = ("cache=cache(), requests=3, rows=7, heads=4, scale=0.1, causal=True, row_offsets=1*M, lengths=2*M, page_table=3*M, table_width=4, "
            "q=4*M, ld_q=256, out=5*M, ld_out=256")
    expected = {"scale=2.3e38": "taken", "scale=-2.3e38": "taken", "scale=2.4e38": "unsupported", "scale=-3.4e38": "unsupported", "scale=1e-45": "taken"}
    assert answers(stub, "hip.attention_kv_cache_bf16_dev", base, expected) == list(expected.values())


def test_results_over_what_is_read(stub):
    """Positions, slots, offsets, lengths and page tables within what a call writes; beside it, and between its rows, they may be."""
    for call, size in (("hip.rotary_f32_dev", 4), ("hip.rotary_bf16_dev", 2)):
        base = "rows=3, heads=2, head_dim=64, rotary=hip.Rotary(64), positions=3*M, src=2*M, ld_in=128, dst=3*M, ld_out=128"
        rows = 3 * 128 * size
        expected = {"": "invalid", "positions=3*M - 8": "invalid", "positions=3*M - 12": "taken", f"positions=3*M + {rows - 4}": "invalid",
                    f"positions=3*M + {rows}": "taken", f"ld_out=200, positions=3*M + {128 * size}": "taken",
                    f"ld_out=200, positions=3*M + {200 * size - 12}": "taken", f"ld_out=200, positions=3*M + {200 * size - 8}": "invalid",
                    f"ld_out=200, positions=3*M + {300 * size}": "invalid", f"ld_out=200, positions=3*M + {328 * size}": "taken",
                    "positions=2*M": "taken", "src=3*M, positions=3*M + 4": "invalid", "positions=None, sequence=2": "taken"}
        assert answers(stub, call, base, expected) == list(expected.values())
    for call in ("hip.kv_cache_append_f32_dev", "hip.kv_cache_append_bf16_dev"):
        base = "cache=cache(), rows=5, slots=1*M, k=2*M, v=3*M, ld=128"
        expected = {"slots=16*M - 16": "invalid", "slots=16*M - 20": "taken", "slots=32*M + 65532": "invalid", "slots=32*M + 65536": "taken",
                    "slots=48*M + 8": "invalid", "slots=64*M + 60": "invalid", "slots=2*M": "taken"}
        assert answers(stub, call, base, expected) == list(expected.values())
    base = ("cache=cache(), requests=3, rows=7, heads=4, scale=0.1, causal=True, row_offsets=1*M, lengths=2*M, page_table=3*M, table_width=4, "
            "q=4*M, ld_q=256, out=5*M, ld_out=256")
    expected = {"out=1*M": "invalid", "out=1*M + 8": "invalid", "out=1*M + 16": "taken", "out=2*M": "invalid", "out=2*M + 16": "taken", "out=3*M + 40": "invalid",
                "out=3*M + 48": "taken", "row_offsets=5*M + 3580": "invalid", "row_offsets=5*M + 3584": "taken", "lengths=5*M - 12": "taken",
                "page_table=5*M - 44": "invalid", "ld_out=512, page_table=5*M + 512": "taken", "ld_out=512, page_table=5*M + 1536": "taken",
                "ld_out=512, page_table=5*M + 1000": "invalid", "table_width=0, page_table=5*M": "taken"}
    assert answers(stub, "hip.attention_kv_cache_bf16_dev", base, expected) == list(expected.values())


def test_attention_goes_on_without_room_for_parts(stub):
    """Long contexts of few rows are cut over workgroups; without scratch memory for the parts, one takes a context as it is."""
    out = run(stub, """
for fail in (1, 0):
    no_memory.value, before = fail, launches.value
    hip.attention_kv_cache_bf16_dev(cache(pages=4000), 1, 1, 4, 0.1, True, M, 2 * M, 3 * M, 2000, 4 * M, 256, 5 * M, 256)
    print(launches.value - before, grid.value)
""")
    assert out[:2] == ["1", "2"] and out[2] == "1" and int(out[3]) > 2
    out = run(stub, """
for fail in (1, 0):
    no_memory.value = fail
    hip.attention_kv_cache_bf16_dev(cache(pages=4000), 1, 300, 4, 0.1, True, M, 2 * M, 3 * M, 2000, 4 * M, 256, 5 * M, 256)
    print(grid.value)
""")
    assert out[0] == "22" and int(out[1]) > 22  # eight narrow tiles of columns and three wide ones, of two heads


def test_contexts_are_cut_among_any_number_of_requests(stub):
    """Two key heads, a narrow tile of columns for each request and one for each sixteen columns, and 512 workgroups more for parts; none more for
    a table of no more keys than a workgroup takes."""
    out = run(stub, """
for requests in (60, 2040, 5000):
    for width in (2000, 4):
        hip.attention_kv_cache_bf16_dev(cache(pages=4000), requests, requests, 4, 0.1, True, M, 2 * M, 2**40, width, 2**41, 256, 2**42, 256)
        print(grid.value - 2 * (requests + requests * 2 // 16))
""")
    assert out == ["512", "0"] * 3


def test_no_parts_where_key_heads_fill_the_chip(stub):
    """A share of as many workgroups as there should be is longer than any context then: nothing is cut, and no memory is kept for parts."""
    out = run(stub, """
memory = ctypes.c_ulonglong.in_dll(stub, "stub_memory_used")
for heads in (512, 513, 5000):
    hip.release_scratch()
    before = memory.value
    c = cache(pages=100, heads=heads, k=2**43, v=2**44, ks=2**45, vs=2**46)
    hip.attention_kv_cache_bf16_dev(c, 1, 1, heads, 0.1, True, M, 2 * M, 2**40, 2000, 2**41, heads * 64, 2**42, heads * 64)
    print(grid.value - heads, memory.value - before > 0)
""")
    assert out == ["512", "True", "0", "False", "0", "False"]


def test_null_structures():
    from spiraltorch_amd import hip
    with pytest.raises(ValueError):
        hip.KvCache(0, 64, 1, 64, 1, 1, 1, 1)
    with pytest.raises(ValueError):
        hip.KvCache(4, 64, -1, 64, 1, 1, 1, 1)
