"""Log-probabilities of given tokens, entropies, the likeliest alternatives and the logits' gradient against 64 bits."""
import numpy as np
import pytest
import torch

from spiraltorch_amd import inputs

pytestmark = pytest.mark.gpu

F, U = 2.0**-24, 2.0**-8
LEAST = 2.0**-126  # the exponential instruction gives no subnormal numbers


def oracle(x, tokens):
    """Of (rows, vocab) values: normalizers, probabilities, log-probabilities of all, entropies, and of the tokens."""
    with np.errstate(divide="ignore", invalid="ignore"):
        most = x.max(1, keepdims=True)
        safe = np.where(np.isfinite(most), most, 0.0)
        lse = (safe + np.log(np.exp(x - safe).sum(1, keepdims=True)))[:, 0]
        log_p = np.where(np.isinf(lse)[:, None], -np.inf, x - np.where(np.isinf(lse), 0.0, lse)[:, None])
    p = np.exp(log_p)
    entropies = -np.where(p > 0, p * np.where(p > 0, log_p, 0.0), 0.0).sum(1)
    counts = (tokens >= 0) & (tokens < x.shape[1])
    log_probs = np.where(counts, log_p[np.arange(len(x)), np.where(counts, tokens, 0)], 0.0)
    return lse, p, log_p, entropies, log_probs, counts


def bounds(x, lse, entropies):
    """How far the normalizer and the entropy may be off.  Every difference from the maximum is off by half a step of it and of its
    product with log2 e, which are as relative errors of its exponential 2 f |x - m| log2 e at the most, and each exponential and its sums by
    some steps; a thread adds up to vocab / 64 + 64 values, then 8 times two sums."""
    finite = np.where(np.isfinite(x), x, np.nan)
    with np.errstate(invalid="ignore"), np.testing.suppress_warnings() as quiet:
        quiet.filter(RuntimeWarning)
        m = np.nan_to_num(np.nanmax(finite, 1))
        terms = x.shape[1] / 64 + 80
        # weights of far values are small: |d| e^-d is at most 1/e of the largest, so that their share counts with |d| up to the row's spread
        spread = np.minimum(np.nan_to_num(m - np.nanmin(finite, 1)), 120.0)
    e_l = (terms + 4 * spread + 8) * F  # relative, of L, and of T's terms
    safe = np.where(np.isfinite(lse), lse, 0.0)
    e_lse = e_l + 2 * F * np.abs(safe) + 4 * F * (1 + np.abs(safe - m))
    e_h = e_l * (2 + 2 * np.abs(safe - m) + spread) + 8 * F * (1 + np.abs(safe - m))
    return e_lse, e_h


def make(rng, rows, ld, kind, spread=3.0):
    x = (spread * rng.normal(size=(rows, ld))).astype(np.float32)
    return x if kind == "f32" else inputs.to_bf16(x)


def floats(x):
    return (x if x.dtype == np.float32 else inputs.from_bf16(x)).astype(np.float64)


class Call:
    def __init__(self, hip, x, vocab, tokens, kind, top=0, offset=0):
        self.hip, self.kind, self.vocab, self.top, self.x, self.offset = hip, kind, vocab, top, x, offset
        self.rows, self.ld = x.shape[0], x.shape[1]
        self.tokens = np.asarray(tokens, np.int32)
        dev = hip.DeviceBuffer.from_array
        self.d_x, self.d_tokens = dev(x), dev(self.tokens)
        self.d = {name: dev(np.full(self.rows, 7, np.float32)) for name in ("log_probs", "entropies", "lse")}
        self.d_ids, self.d_top = dev(np.full(max(1, self.rows * top), 7, np.int32)), dev(np.full(max(1, self.rows * top), 7, np.float32))

    def at(self):
        return self.d_x.at(self.offset * self.x.itemsize)

    def forward(self, stream=None):
        call = self.hip.token_log_probs_f32_dev if self.kind == "f32" else self.hip.token_log_probs_bf16_dev
        call(self.rows, self.vocab, self.at(), self.ld, self.d_tokens, self.d["log_probs"], self.d["entropies"], self.d["lse"], self.top,
             self.d_ids if self.top else None, self.d_top if self.top else None, stream=stream)

    def results(self):
        self.hip.device_synchronize()
        r = {name: buf.to_array(np.float32, self.rows) for name, buf in self.d.items()}
        r["ids"] = self.d_ids.to_array(np.int32, (self.rows, self.top))
        r["top"] = self.d_top.to_array(np.float32, (self.rows, self.top))
        return r

    def values(self):
        return floats(self.x)[:, self.offset:self.offset + self.vocab]

    def check(self, what=""):
        self.forward()
        got, x = self.results(), self.values()
        lse, p, log_p, entropies, log_probs, counts = oracle(x, self.tokens)
        e_lse, e_h = bounds(x, lse, entropies)

        def close(a, want, bound, name):
            a = a.astype(np.float64)
            with np.errstate(invalid="ignore"):
                off = np.where(a == want, 0.0, np.abs(a - want))
            assert (off <= np.where(np.isfinite(want), bound, 0.0)).all(), f"{what} {name}: off by {off.max():.3e}, {(off > bound).sum()} of {off.size}"

        close(got["lse"], lse, e_lse, "normalizers")
        close(got["entropies"], entropies, e_h, "entropies")
        close(got["log_probs"], log_probs, e_lse + F * np.abs(np.where(np.isfinite(log_probs), log_probs, 0.0)), "log_probs")
        if self.top:
            ids = np.argsort(-x, 1, kind="stable")[:, :self.top]
            assert (got["ids"] == ids).all(), f"{what} alternatives"
            want = np.take_along_axis(log_p, ids, 1)
            close(got["top"], want, e_lse[:, None] + F * np.abs(np.where(np.isfinite(want), want, 0.0)), "their log_probs")
        return got


SIZES = [(1, 1), (3, 2), (5, 7), (1, 63), (2, 64), (7, 65), (4, 255), (9, 256), (3, 1000), (2, 1025), (1, 2047), (2, 2049), (5, 4097), (1, 8191), (3, 20011),
         (1, 65536), (2, 100001), (1, 262144)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_sizes(hip, rows, vocab, top, kind):
    rng = np.random.default_rng(rows + vocab)
    x = make(rng, rows, vocab, kind)
    Call(hip, x, vocab, rng.integers(0, vocab, rows), kind, min(top, vocab)).check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [50, 1500, 30000])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_rows_at_any_boundary(hip, kind, vocab, offset):
    rng = np.random.default_rng(vocab + offset)
    x = make(rng, 5, vocab + 9, kind)
    Call(hip, x, vocab, rng.integers(0, vocab, 5), kind, 6, offset).check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 5000, 70000])
@pytest.mark.parametrize("shape", ["equal", "rising", "falling", "two values", "late", "barred", "signed zeros"])
def test_orders_and_ties(hip, kind, vocab, shape):
    rng = np.random.default_rng(vocab)
    x = {"equal": np.full((2, vocab), 1.5), "rising": np.tile(np.arange(vocab) / 64.0, (2, 1)), "falling": np.tile(-np.arange(vocab) / 64.0, (2, 1)),
         "two values": rng.integers(0, 2, (2, vocab)) * 0.25, "late": np.where(np.arange(vocab) >= vocab - 40, 3.0, rng.normal(size=(2, vocab))),
         "barred": np.where(rng.random((2, vocab)) < 0.999, -np.inf, rng.normal(size=(2, vocab))),
         "signed zeros": np.where(rng.random((2, vocab)) < 0.5, -0.0, 0.0)}[shape].astype(np.float32)
    x[:, 7] = np.maximum(x[:, 7], 0.0)
    for top in (1, 20, 32):
        Call(hip, x if kind == "f32" else inputs.to_bf16(x), vocab, [7, 7], kind, top).check(f"{shape} {top}")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [100, 40000])
def test_special_rows(hip, kind, vocab):
    """A row of -infinity, of the type's lowest value, with NaN, with +infinity, tokens that do not count, a barred token."""
    rng = np.random.default_rng(3)
    lowest = np.finfo(np.float32).min if kind == "f32" else inputs.from_bf16(np.array([0xFF7F], np.uint16))[0]
    x = rng.normal(size=(8, vocab)).astype(np.float32)
    x[0] = -np.inf
    x[1] = lowest
    x[2, 5] = np.nan
    x[3, 6] = np.inf
    x[4, 10:] = lowest
    x[6, 9] = -np.inf
    call = Call(hip, x if kind == "f32" else inputs.to_bf16(x), vocab, [1, 1, 1, 1, 1, -1, 9, vocab], kind, 3)
    call.forward()
    got = call.results()
    assert got["lse"][0] == -np.inf and got["entropies"][0] == 0 and got["log_probs"][0] == -np.inf
    assert got["ids"][0].tolist() == [0, 1, 2] and (got["top"][0] == -np.inf).all()
    assert abs(got["entropies"][1] - np.log(vocab)) < 1e-5 and got["lse"][1] == lowest  # log(vocab) is nothing beside it
    for row in (2, 3):
        assert np.isnan(got["lse"][row]) and np.isnan(got["entropies"][row]) and np.isnan(got["log_probs"][row])
    assert 5 not in got["ids"][2] and got["log_probs"][5] == 0 and got["log_probs"][7] == 0 and got["log_probs"][6] == -np.inf
    rows = [4, 5, 6, 7]
    lse, _, _, entropies, _, _ = oracle(call.values()[rows], call.tokens[rows])
    assert np.abs(got["lse"][rows] - lse).max() < 1e-5 and np.abs(got["entropies"][rows] - entropies).max() < 1e-4


def gradient(x, tokens, g, h):
    lse, p, log_p, entropies, _, counts = oracle(x, tokens)
    one = np.zeros_like(p)
    one[np.arange(len(x))[counts], tokens[counts]] = 1.0
    g, h = np.where(counts, g, 0.0)[:, None], h[:, None]
    with np.errstate(invalid="ignore"):
        inner = np.where(p > 0, log_p + entropies[:, None], 0.0)
    return g * (one - p) - h * p * inner, p * (np.abs(g) + np.abs(h) * (np.abs(inner) + 1)), np.abs(g) * one


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("with_entropies", [False, True])
@pytest.mark.parametrize("rows,vocab,offset,extra", [(1, 1, 0, 0), (3, 2, 0, 0), (5, 300, 0, 0), (5, 301, 1, 7), (2, 2048, 0, 8), (3, 5001, 0, 0), (4, 5001, 3, 6),
                                                     (1, 100001, 0, 0), (600, 50, 0, 0), (2, 65536, 0, 0)])
def test_gradients(hip, rows, vocab, offset, extra, with_entropies, kind):
    rng = np.random.default_rng(rows * 7 + vocab)
    x = make(rng, rows, vocab + extra + offset, kind)
    x[0, offset:offset + vocab // 3] = -np.inf if kind == "f32" else 0xFF80
    tokens = rng.integers(0, vocab, rows)
    tokens[rows // 2] = -1
    call = Call(hip, x, vocab, tokens, kind, offset=offset)
    call.forward()
    got = call.results()
    g, h = rng.normal(size=rows).astype(np.float32), rng.normal(size=rows).astype(np.float32)
    if not with_entropies:
        h[:] = 0
    d_g, d_h = hip.DeviceBuffer.from_array(g), hip.DeviceBuffer.from_array(h)
    backward = hip.token_log_probs_backward_f32_dev if kind == "f32" else hip.token_log_probs_backward_bf16_dev
    want, size, one = gradient(call.values(), call.tokens, g.astype(np.float64), h.astype(np.float64))
    lse, _, _, entropies, _, _ = oracle(call.values(), call.tokens)
    e_lse, e_h = bounds(call.values(), lse, entropies)
    spread = np.abs(np.where(np.isfinite(call.values()), call.values(), 0.0)) + np.abs(np.where(np.isfinite(lse), lse, 0))[:, None]
    relative = e_lse[:, None] + 4 * F * spread + 16 * F
    bound = size * (relative + e_h[:, None]) + 4 * F * (np.abs(want) + one) + LEAST * (1 + np.abs(g) + np.abs(h))[:, None] * 200
    if kind == "bf16":
        bound += U * (np.abs(want) + bound) + 2.0**-133
    for where in ("beside", "other stride", "in place"):
        if where == "in place":
            d_y, ld_y, at, before = call.d_x, call.ld, call.at(), x
        else:
            ld_y = call.ld if where == "beside" else vocab + 3
            before = np.full((rows, ld_y), 7, x.dtype)
            d_y = hip.DeviceBuffer.from_array(before)
            at = d_y.at(offset * x.itemsize if where == "beside" else 0)
        backward(rows, vocab, call.at(), call.ld, call.d_tokens, call.d["lse"], call.d["entropies"] if with_entropies else None, d_g,
                 d_h if with_entropies else None, at, ld_y)
        hip.device_synchronize()
        all_of = d_y.to_array(x.dtype, (rows, ld_y))
        first = 0 if where == "other stride" else offset
        y = floats(all_of)[:, first:first + vocab]
        off = np.abs(y - want)
        assert (off <= bound).all(), f"{where}: {(off > bound).sum()} of {off.size} outside, worst {np.max(off / np.maximum(bound, 1e-300)):.2f} of the bound"
        beside = np.ones(all_of.shape, bool)
        beside[:, first:first + vocab] = False
        assert (all_of[beside] == before[beside]).all(), f"{where}: values beside the rows"


def test_gradient_of_nothing(hip):
    """A row of -infinity has the gradient 0; without gradients given, all of it is 0."""
    x = np.full((2, 100), -np.inf, np.float32)
    x[1] = 1.0
    call = Call(hip, x, 100, [3, 3], "f32")
    call.forward()
    d_g, d_y = hip.DeviceBuffer.from_array(np.ones(2, np.float32)), hip.DeviceBuffer.from_array(np.full((2, 100), 7, np.float32))
    hip.token_log_probs_backward_f32_dev(2, 100, call.d_x, 100, call.d_tokens, call.d["lse"], call.d["entropies"], d_g, d_g, d_y, 100)
    hip.device_synchronize()
    y = d_y.to_array(np.float32, (2, 100))
    assert (y[0] == 0).all() and abs(y[1, 3] - 0.99) < 1e-5
    hip.token_log_probs_backward_f32_dev(2, 100, call.d_x, 100, None, call.d["lse"], None, None, None, d_y, 100)
    hip.device_synchronize()
    assert (d_y.to_array(np.float32, (2, 100)) == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_far_into_the_memory(hip, kind):
    """Logits of 9 GB: the last rows' results, and gradients, are those that they have alone."""
    rng = np.random.default_rng(4)
    size = 4 if kind == "f32" else 2
    vocab, rows = 60001, 9 * 10**9 // size // 60001
    x = make(rng, 3, vocab, kind)
    tokens, g = rng.integers(0, vocab, 3).astype(np.int32), rng.normal(size=3).astype(np.float32)
    alone = Call(hip, x, vocab, tokens, kind, 4)
    alone.forward()
    want = alone.results()
    backward = hip.token_log_probs_backward_f32_dev if kind == "f32" else hip.token_log_probs_backward_bf16_dev
    d_g, d_y = hip.DeviceBuffer.from_array(g), hip.DeviceBuffer(3 * vocab * size)
    backward(3, vocab, alone.d_x, vocab, alone.d_tokens, alone.d["lse"], alone.d["entropies"], d_g, d_g, d_y, vocab)
    hip.device_synchronize()
    want_y = d_y.to_array(x.dtype, x.shape)
    d_x = hip.DeviceBuffer(rows * vocab * size)
    d_x.zero()
    d_x.upload(x, (rows - 3) * vocab * size)
    d_tokens = hip.DeviceBuffer.from_array(np.concatenate([np.zeros(rows - 3, np.int32), tokens]))
    d_all = hip.DeviceBuffer.from_array(np.concatenate([np.zeros(rows - 3, np.float32), g]))
    out = [hip.DeviceBuffer(rows * 4) for _ in range(3)]
    d_ids, d_top = hip.DeviceBuffer(rows * 16), hip.DeviceBuffer(rows * 16)
    forward = hip.token_log_probs_f32_dev if kind == "f32" else hip.token_log_probs_bf16_dev
    forward(rows, vocab, d_x, vocab, d_tokens, *out, 4, d_ids, d_top)
    hip.device_synchronize()
    got = {name: buf.to_array(np.float32, rows)[-3:] for name, buf in zip(("log_probs", "entropies", "lse"), out)}
    for name, value in got.items():
        # (few rows are cut into parts, whose sums are put together in another order)
        assert np.abs(value - want[name]).max() < 1e-4, name
    assert (d_ids.to_array(np.int32, (rows, 4))[-3:] == want["ids"]).all()
    backward(rows, vocab, d_x, vocab, d_tokens, out[2], out[1], d_all, d_all, d_x, vocab)
    hip.device_synchronize()
    y = np.empty((3, vocab), x.dtype)
    hip._check(hip._lib.load().st_hip_memcpy_d2h(y.ctypes.data, d_x.at((rows - 3) * vocab * size), y.nbytes, None))
    off = np.abs(floats(y) - floats(want_y))
    assert (off <= 2e-4 * np.abs(floats(want_y)) + (U * np.abs(floats(want_y)) * 2 if kind == "bf16" else 0) + 1e-9).all()


def test_the_same_bits_again(hip):
    rng = np.random.default_rng(8)
    for rows, vocab in ((1, 100000), (70, 30000), (500, 700)):
        call = Call(hip, make(rng, rows, vocab, "bf16"), vocab, rng.integers(0, vocab, rows), "bf16", 16)
        call.forward()
        first = call.results()
        for _ in range(3):
            call.forward()
            for name, value in call.results().items():
                assert (value == first[name]).all(), name


def test_parts_captured_and_replayed(hip):
    """A row that is cut into parts, recorded on a stream without scratch memory."""
    x = torch.randn(2, 90000, device="cuda")
    tokens = torch.tensor([5, 89999], dtype=torch.int32, device="cuda")
    out = [torch.empty(2, device="cuda") for _ in range(3)]
    ids, top = torch.empty(2, 9, dtype=torch.int32, device="cuda"), torch.empty(2, 9, device="cuda")
    call = lambda stream: hip.token_log_probs_f32_dev(2, 90000, x.data_ptr(), 90000, tokens.data_ptr(), *(o.data_ptr() for o in out), 9, ids.data_ptr(),
                                                      top.data_ptr(), stream=stream)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        call(torch.cuda.current_stream().cuda_stream)
    try:
        for replay in range(4):
            x.mul_(-0.9)
            call(None)
            torch.cuda.synchronize()
            want = [o.clone() for o in (*out, ids, top)]
            for o in (*out, ids, top):
                o.fill_(7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            for got, first in zip((*out, ids, top), want):
                assert torch.equal(got, first), replay
    finally:
        del graph
        hip.release_scratch(stream.cuda_stream)
        hip.release_scratch(None)


@pytest.mark.parametrize("vocab", [2, 4, 40, 5001])
def test_the_entropy_goes_with_the_normalizer(hip, vocab):
    """The gradient of the entropy sums to 0 over a row to its own terms' rounding, also where one token has nearly all: there log p + H is small beside
    what the normalizer's rounding moves log p by (half a step of 8 to 16: 8 f), which the entropy moves with."""
    rng = np.random.default_rng(vocab)
    rows = 64
    x = rng.normal(size=(rows, vocab)).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    x[np.arange(rows), tokens] += 10.0 + np.log(vocab)
    x = np.minimum(x, 15.0).astype(np.float32) if vocab < 100 else x
    call = Call(hip, x, vocab, tokens, "f32")
    call.check()
    ones, d_y = hip.DeviceBuffer.from_array(np.ones(rows, np.float32)), hip.DeviceBuffer.from_array(np.zeros((rows, vocab), np.float32))
    hip.token_log_probs_backward_f32_dev(rows, vocab, call.at(), call.ld, call.d_tokens, call.d["lse"], call.d["entropies"], None, ones, d_y, vocab)
    hip.device_synchronize()
    y = d_y.to_array(np.float32, (rows, vocab)).astype(np.float64)
    lse, p, log_p, entropies, _, _ = oracle(call.values(), call.tokens)
    assert (np.abs(lse) < 32).all()
    # a term: p's exponent rounded twice (2 f |log p| each) and its result, log p and H and their sum rounded, the product twice; and H, the sum of
    # what up to vocab / 64 + 80 additions leave of T / L
    size = (p * (np.abs(log_p) + entropies[:, None]) * (8 + 4 * np.abs(log_p))).sum(1) + (vocab / 64 + 80 + 4 * 40) * entropies
    assert (np.abs(y.sum(1)) <= F * size).all(), np.max(np.abs(y.sum(1)) / (F * size))
