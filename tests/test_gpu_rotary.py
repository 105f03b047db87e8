"""Rotary positions against the formula in 64 bits."""
import numpy as np
import pytest

import paged_cache_oracle as plain
from spiraltorch_amd import inputs

pytestmark = pytest.mark.gpu

# cos and sin: the angle's rounding (less than one half step of 1), the functions (at most two) and the magnitude; then two products and
# a sum: eight half steps of |a| + |b| hold them all.  A value of bf16 is rounded once more.
F32_STEPS, BF16_STEP = 8 * 2.0**-24, 2.0**-8


def run(hip, x, ld_in, heads, dim, config, positions, ld_out, offset=0, **options):
    """x: (rows, ld_in) of the type; the head block begins `offset` values into a row.  Returns (rows, ld_out) with sentinels where nothing was
    written."""
    rows, size = x.shape[0], x.itemsize
    src = hip.DeviceBuffer.from_array(x)
    sentinel = np.full((rows, ld_out), 7, x.dtype)
    dst = hip.DeviceBuffer.from_array(sentinel)
    d_pos = None if positions is None else hip.DeviceBuffer.from_array(np.asarray(positions, np.int32))
    call = hip.rotary_f32_dev if x.dtype == np.float32 else hip.rotary_bf16_dev
    call(rows, heads, dim, hip.Rotary(**config), d_pos, src.at(offset * size), ld_in, dst, ld_out, **options)
    hip.device_synchronize()
    return dst.to_array(x.dtype, (rows, ld_out)), src.to_array(x.dtype, x.shape)


def floats(a):
    return a.astype(np.float64) if a.dtype == np.float32 else inputs.from_bf16(a).astype(np.float64)


def make(rng, shape, kind):
    x = rng.normal(size=shape).astype(np.float32)
    return x if kind == "f32" else inputs.to_bf16(x)


def check(got, x, heads, dim, config, positions, transposed, kind, what):
    config = dict(config)
    turned, interleaved, magnitude = config.pop("rotary_dim"), config.pop("interleaved", False), config.pop("magnitude", 1.0)
    # the configuration's numbers are f32
    per = plain.turns(turned, **{name: float(np.float32(value)) for name, value in config.items()})
    want, size = plain.rotary(floats(x).reshape(-1, heads, dim), positions, turned, interleaved, per, float(np.float32(magnitude)), transposed)
    bound = F32_STEPS * size + (BF16_STEP * np.abs(want) if kind == "bf16" else 0)
    bound[..., turned:] = 0.0  # copied
    err = np.abs(floats(got).reshape(want.shape) - want)
    assert (err <= bound).all(), f"{what}: {(err > bound).sum()} of {err.size} outside, worst {np.max(err - bound):.3e}"


CASES = [
    # rows, heads, dim, rotary_dim, extra columns, options
    (1, 1, 2, 2, 0, {}), (1, 1, 64, 64, 0, {}), (3, 5, 64, 32, 0, {}), (17, 3, 80, 80, 0, {}), (4, 40, 128, 128, 1024, {"base": 500000.0}),
    (5, 2, 256, 64, 8, {"factor": 4.0}), (33, 7, 96, 24, 0, {"magnitude": 1.25}), (2, 3, 10, 6, 3, {}), (7, 1, 130, 130, 1, {}),
    (130, 4, 64, 64, 64, {"base": 500000.0, "factor": 8.0, "original_length": 8192.0}),
    (9, 6, 128, 96, 16, {"factor": 2.5, "original_length": 4096.0, "low_turns": 1.0, "high_turns": 32.0, "magnitude": 0.7}),
    (2, 1, 1024, 1024, 0, {}), (6, 2, 64, 0, 0, {}), (1000, 3, 128, 128, 0, {}), (3, 70, 48, 16, 0, {}), (5, 1, 72, 36, 4, {}),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,turned,extra,options", CASES)
def test_against_the_formula(hip, rows, heads, dim, turned, extra, options, interleaved, kind):
    rng = np.random.default_rng(rows * 1000 + dim + turned + interleaved)
    config = {"rotary_dim": turned, "interleaved": interleaved, **options}
    width = heads * dim
    x = make(rng, (rows, width + extra), kind)
    positions = rng.integers(0, 4096, rows)
    positions[0] = 0
    got, after = run(hip, x, width + extra, heads, dim, config, positions, width + 2 * extra)
    assert (after == x).all()
    assert (got[:, width:] == 7).all(), "columns behind the heads"
    check(got[:, :width], x[:, :width], heads, dim, config, positions, False, kind, "forward")
    got, _ = run(hip, x, width + extra, heads, dim, config, positions, width, transposed=True)
    check(got, x[:, :width], heads, dim, config, positions, True, kind, "transposed")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_far_and_negative_positions(hip, kind):
    positions = [0, 1, -1, 131071, 1048576, 10**7 + 1, -(10**6), 2**31 - 1, -(2**31)]
    config = {"rotary_dim": 128, "base": 10000.0}
    x = make(np.random.default_rng(2), (len(positions), 2 * 128), kind)
    got, _ = run(hip, x, 256, 2, 128, config, positions, 256)
    check(got, x, 2, 128, config, positions, False, kind, "far positions")


@pytest.mark.parametrize("dim,turned,offset", [(64, 64, 1), (64, 64, 4), (64, 32, 8), (96, 96, 2), (128, 128, 0)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_unaligned_rows_and_strides(hip, kind, dim, turned, offset):
    rng = np.random.default_rng(offset + dim)
    x = make(rng, (6, 3 * dim + 5), kind)
    positions = rng.integers(0, 500, 6)
    for interleaved in (False, True):
        config = {"rotary_dim": turned, "interleaved": interleaved}
        got, _ = run(hip, x[:, :], 3 * dim + 5, 2, dim, config, positions, 2 * dim + 1, offset=offset)
        flat = np.stack([row[offset:offset + 2 * dim] for row in x])
        check(got[:, :2 * dim], flat, 2, dim, config, positions, False, kind, "unaligned")
        assert (got[:, 2 * dim:] == 7).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved,dim,turned", [(False, 64, 64), (True, 128, 32), (False, 80, 20), (True, 6, 4)])
def test_in_place_and_between_columns_of_one_matrix(hip, kind, interleaved, dim, turned):
    """Queries and keys of a fused projection turned where they are: the values stay; and from one block of columns into another."""
    rng = np.random.default_rng(dim + turned)
    rows, heads = 21, 3
    x = make(rng, (rows, 2 * heads * dim), kind)
    positions = rng.integers(0, 9000, rows)
    config = {"rotary_dim": turned, "interleaved": interleaved}
    call = hip.rotary_f32_dev if kind == "f32" else hip.rotary_bf16_dev
    buf, d_pos = hip.DeviceBuffer.from_array(x), hip.DeviceBuffer.from_array(positions.astype(np.int32))
    width = heads * dim
    call(rows, heads, dim, hip.Rotary(**config), d_pos, buf, 2 * width, buf, 2 * width)
    hip.device_synchronize()
    got = buf.to_array(x.dtype, x.shape)
    assert (got[:, width:] == x[:, width:]).all()
    check(got[:, :width], x[:, :width], heads, dim, config, positions, False, kind, "in place")
    buf.upload(x)
    call(rows, heads, dim, hip.Rotary(**config), d_pos, buf, 2 * width, buf.at(width * x.itemsize), 2 * width)
    hip.device_synchronize()
    got = buf.to_array(x.dtype, x.shape)
    assert (got[:, :width] == x[:, :width]).all()
    check(got[:, width:], x[:, :width], heads, dim, config, positions, False, kind, "into other columns")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,dim,turned", [(3000, 14, 96, 36), (2500, 9, 65, 22), (5000, 12, 80, 40)])
def test_many_rows_of_short_runs(hip, kind, rows, heads, dim, turned):
    """Runs of two values, one and four, where a thread has several at once."""
    rng = np.random.default_rng(rows)
    x = make(rng, (rows, heads * dim), kind)
    positions = rng.integers(0, 3000, rows)
    for interleaved in (False, True):
        config = {"rotary_dim": turned, "interleaved": interleaved}
        got, _ = run(hip, x, heads * dim, heads, dim, config, positions, heads * dim)
        check(got, x, heads, dim, config, positions, False, kind, f"interleaved {interleaved}")


def test_positions_from_the_row(hip):
    x = make(np.random.default_rng(4), (3 * 37, 64), "f32")
    config = {"rotary_dim": 64, "interleaved": True}
    got, _ = run(hip, x, 64, 1, 64, config, None, 64, sequence=37)
    check(got, x, 1, 64, config, np.arange(3 * 37) % 37, False, "f32", "row % sequence")


def test_the_gradient_is_the_transpose(hip):
    """<turn(x), g> = <x, transposed(g)> in 64 bits, and the difference quotient of a weighted sum along a direction: the map is linear, so
    that it is the derivative whatever the step."""
    rng = np.random.default_rng(8)
    config = {"rotary_dim": 48, "interleaved": False, "magnitude": 1.1}
    x, g = make(rng, (50, 4 * 64), "f32"), make(rng, (50, 4 * 64), "f32")
    positions = rng.integers(0, 3000, 50)
    y, _ = run(hip, x, 256, 4, 64, config, positions, 256)
    gx, _ = run(hip, g, 256, 4, 64, config, positions, 256, transposed=True)
    left, right = np.sum(floats(y) * floats(g)), np.sum(floats(x) * floats(gx))
    room = 2 * F32_STEPS * 2.2 * (np.abs(floats(x)).sum() * np.abs(floats(g)).max() + np.abs(floats(g)).sum() * np.abs(floats(x)).max())
    assert abs(left - right) <= room
    direction = make(rng, (50, 4 * 64), "f32")
    step = 0.5
    moved, _ = run(hip, (x + np.float32(step) * direction).astype(np.float32), 256, 4, 64, config, positions, 256)
    numeric = np.sum((floats(moved) - floats(y)) / step * floats(g))
    assert abs(numeric - np.sum(floats(gx) * floats(direction))) <= 10 * room


def test_special_values_stay_in_their_pair(hip):
    x = np.ones((2, 64), np.float32)
    x[0, 3], x[1, 40] = np.nan, np.inf
    got, _ = run(hip, x, 64, 1, 64, {"rotary_dim": 64}, [5, 0], 64)
    bad = ~np.isfinite(got)
    assert set(map(tuple, np.argwhere(bad))) <= {(0, 3), (0, 35), (1, 8), (1, 40)} and bad[0, 3] and bad[1, 40]


def test_nothing_to_do(hip):
    config = hip.Rotary(64)
    hip.rotary_f32_dev(0, 4, 64, config, None, None, 256, None, 256, sequence=1)
    hip.rotary_bf16_dev(5, 0, 64, config, None, None, 0, None, 0, sequence=1)
