"""Attention that is trained, in bf16: its forward and its backward pass against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

import training_oracle as plain
from spiraltorch_amd import inputs

pytestmark = pytest.mark.gpu

SENTINEL = 0x4567


class Case:
    """Buffers of one call, on the device: matrices with columns of their own and columns beside them that stay as they are."""

    def __init__(self, hip, seed, batch, heads, kv_heads, n, dim, causal=False, lengths=None, scale=None, buckets=0, far=0, extra=0, spread=1.0,
                 bidirectional=None):
        rng = np.random.default_rng(seed)
        self.hip, self.shape = hip, (batch, heads, kv_heads, n, dim)
        self.causal, self.lengths, self.scale, self.far = causal, lengths, dim**-0.5 if scale is None else scale, far
        self.bidirectional = not causal if bidirectional is None else bidirectional
        rows, width, kv = batch * n, heads * dim, kv_heads * dim
        self.ld_qkv, self.ld_out = width + 2 * kv + extra, width + extra
        make = lambda *shape: inputs.to_bf16((spread * rng.normal(size=shape)).astype(np.float32))
        self.qkv, self.g = make(rows, self.ld_qkv), make(rows, self.ld_out)
        self.table = rng.normal(size=(buckets, heads)).astype(np.float32) if buckets else None
        dev = hip.DeviceBuffer.from_array
        self.d_qkv, self.d_g = dev(self.qkv), dev(self.g)
        self.d_lengths = None if lengths is None else dev(np.asarray(lengths, np.int32))
        self.d_table = None if self.table is None else dev(self.table)
        self.d_out, self.d_gqkv = dev(np.full((rows, self.ld_out), SENTINEL, np.uint16)), dev(np.full((rows, self.ld_qkv), SENTINEL, np.uint16))
        self.d_lse = dev(np.full(batch * heads * n, 7, np.float32))
        self.d_gtable = None if self.table is None else dev(np.full((buckets, heads), 7, np.float32))
        bias = None if self.table is None else hip.PositionBias(buckets, far, self.d_table, bidirectional=self.bidirectional)
        self.plan = hip.AttentionTraining(batch, heads, n, dim, self.scale, causal=causal, kv_heads=kv_heads, lengths=self.d_lengths, position_bias=bias)

    def forward(self, stream=None):
        batch, heads, kv_heads, n, dim = self.shape
        k, v = 2 * heads * dim, 2 * (heads + kv_heads) * dim
        self.hip.attention_training_bf16_dev(self.plan, self.d_qkv, self.ld_qkv, self.d_qkv.at(k), self.d_qkv.at(v), self.ld_qkv, self.d_out, self.ld_out,
                                             self.d_lse, stream=stream)

    def backward(self, stream=None):
        batch, heads, kv_heads, n, dim = self.shape
        k, v = 2 * heads * dim, 2 * (heads + kv_heads) * dim
        self.hip.attention_backward_bf16_dev(self.plan, self.d_qkv, self.ld_qkv, self.d_qkv.at(k), self.d_qkv.at(v), self.ld_qkv, self.d_out, self.ld_out,
                                             self.d_lse, self.d_g, self.ld_out, self.d_gqkv, self.ld_qkv, self.d_gqkv.at(k), self.d_gqkv.at(v),
                                             self.ld_qkv, self.d_gtable, stream=stream)

    def split(self, x):
        batch, heads, kv_heads, n, dim = self.shape
        x = inputs.from_bf16(x).astype(np.float64).reshape(batch, n, -1)
        a, b, c = heads * dim, (heads + kv_heads) * dim, (heads + 2 * kv_heads) * dim
        return (x[..., :a].reshape(batch, n, heads, dim), x[..., a:b].reshape(batch, n, kv_heads, dim), x[..., b:c].reshape(batch, n, kv_heads, dim))

    def results(self):
        self.hip.device_synchronize()
        batch, heads, kv_heads, n, dim = self.shape
        out, gqkv = self.d_out.to_array(np.uint16, (batch * n, self.ld_out)), self.d_gqkv.to_array(np.uint16, (batch * n, self.ld_qkv))
        assert (out[:, heads * dim:] == SENTINEL).all() and (gqkv[:, (heads + 2 * kv_heads) * dim:] == SENTINEL).all(), "columns beside"
        dq, dk, dv = self.split(gqkv)
        r = {"out": inputs.from_bf16(out[:, :heads * dim]), "lse": self.d_lse.to_array(np.float32, (batch, heads, n)), "dq": dq, "dk": dk, "dv": dv}
        if self.table is not None:
            r["dtable"] = self.d_gtable.to_array(np.float32, self.table.shape)
        return r

    def wanted(self):
        batch, heads, kv_heads, n, dim = self.shape
        q, k, v = self.split(self.qkv)
        g = inputs.from_bf16(self.g).astype(np.float64)[:, :heads * dim].reshape(batch, n, heads, dim)
        table = None if self.table is None else self.table.astype(np.float64)
        return plain.training(q, k, v, g, float(np.float32(self.scale)), self.causal, self.lengths, table, self.far, self.bidirectional)

    def check(self, what=""):
        self.forward()
        self.backward()
        got, want = self.results(), self.wanted()
        for name in want:
            plain.check(got[name], want[name], f"{what} {name}")
        return got


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 257])
def test_lengths(hip, n, causal, dim):
    Case(hip, n + dim, 2, 2, 2, n, dim, causal).check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (6, 2), (7, 7), (8, 4), (10, 2)])
def test_shared_heads(hip, heads, kv_heads, causal, dim):
    Case(hip, heads, 3, heads, kv_heads, 70, dim, causal, extra=8).check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batches(hip, causal, dim):
    """Lengths of 0, of 1, in the middle of a tile, at its end and whole; -3 counts as 0 and 1000 as all."""
    lengths = [0, 1, 37, 64, 128, 129, 200, -3, 1000]
    for buckets in (0, 8):
        Case(hip, 5, len(lengths), 2, 1, 200, dim, causal, lengths=lengths, buckets=buckets, far=20, extra=16).check(f"buckets {buckets}")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bidirectional,causal", [(True, False), (False, True), (False, False), (True, True)])
@pytest.mark.parametrize("buckets,far,n", [(4, 3, 40), (32, 128, 300), (32, 128, 60), (8, 16, 129), (64, 300, 200), (256, 2048, 131), (6, 5, 200)])
def test_position_bias(hip, buckets, far, n, bidirectional, causal, dim):
    Case(hip, buckets + n, 2, 3, 1, n, dim, causal, buckets=buckets, far=far, bidirectional=bidirectional).check()


@pytest.mark.parametrize("causal", [False, True])
def test_far_blocks_of_distances(hip, causal):
    """Whole blocks beyond the last bucket's distance, on both sides."""
    Case(hip, 3, 1, 2, 2, 700, 64, causal, lengths=[690], buckets=16, far=40).check()


def test_buckets_barred_by_minus_infinity(hip):
    """A bias of -infinity bars its bucket; rows that are left with nothing are 0, and so are their gradients."""
    for causal in (False, True):
        case = Case(hip, 9, 1, 2, 2, 100, 64, causal, buckets=8, far=20)
        case.table[1, 0] = -np.inf  # one bucket of the first head
        case.table[:, 1] = -np.inf  # the second head sees nothing
        case.d_table.upload(case.table)
        got = case.check(f"causal {causal}")
        assert (got["lse"][0, 1] == -np.inf).all() and (got["dq"][:, :, 1] == 0).all() and (got["dtable"][:, 1] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0, 1e-20])
@pytest.mark.parametrize("buckets", [0, 8])
def test_scales(hip, scale, buckets):
    Case(hip, 2, 2, 2, 2, 90, 64, True, scale=scale, buckets=buckets, far=30).check()


@pytest.mark.parametrize("dim", [64, 128])
def test_sharp_rows(hip, dim):
    """Scores of some hundred: one key has all the weight."""
    Case(hip, 4, 2, 2, 2, 150, dim, False, spread=6.0).check()


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_behind_a_length_is_not_read(hip, dim):
    lengths = [40, 0, 130]
    for causal in (False, True):
        case = Case(hip, 8, 3, 2, 1, 140, dim, causal, lengths=lengths, buckets=8, far=20)
        clean = case.check()
        for b, m in enumerate(lengths):
            case.qkv[b * 140 + m:(b + 1) * 140] = 0x7FC0  # NaN
            case.g[b * 140 + m:(b + 1) * 140] = 0xFF80  # -infinity
        case.d_qkv.upload(case.qkv)
        case.d_g.upload(case.g)
        case.forward()
        case.backward()
        for name, value in case.results().items():
            assert (value == clean[name]).all(), name


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,n,buckets", [(4, 1, 520, 0), (8, 2, 300, 8), (3, 3, 1100, 0), (7, 1, 260, 12)])
def test_keys_of_few_tiles(hip, heads, kv_heads, n, buckets, causal, dim):
    """Tiles of keys whose rows are cut over workgroups: the parts go through scratch memory; short and empty sequences among them."""
    Case(hip, n + heads, 3, heads, kv_heads, n, dim, causal, lengths=[n, 0, n // 2 + 3], buckets=buckets, far=40, extra=8).check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_the_same_bits_again_and_in_any_batch(hip, causal, dim):
    """Results do not depend on the order of workgroups, nor, where keys are not cut into parts, a sequence's on the others of its batch (whose order is
    that of their lengths)."""
    lengths = [150, 3, 200, 77, 200, 128, 10, 64, 199]
    case = Case(hip, 11, len(lengths), 2, 1, 200, dim, causal, lengths=lengths, buckets=8, far=30)
    case.forward()
    case.backward()
    first = case.results()
    case.forward()
    case.backward()
    for name, value in case.results().items():
        assert (value == first[name]).all(), name
    for b in (0, 2, 8):
        alone = Case(hip, 11, 1, 2, 1, 200, dim, causal, lengths=[lengths[b]], buckets=8, far=30)
        alone.qkv, alone.g, alone.table = case.qkv[b * 200:(b + 1) * 200], case.g[b * 200:(b + 1) * 200], case.table
        for buf, values in ((alone.d_qkv, alone.qkv), (alone.d_g, alone.g), (alone.d_table, alone.table)):
            buf.upload(values)
        alone.forward()
        alone.backward()
        got = alone.results()
        for name in ("out", "dq", "dk", "dv"):
            assert (got[name].reshape(-1) == first[name].reshape(len(lengths), -1)[b]).all(), (b, name)
        assert (got["lse"][0] == first["lse"][b]).all()


def test_more_sequences_than_are_sorted(hip):
    """Beyond 64 sequences they are taken as they come."""
    rng = np.random.default_rng(5)
    Case(hip, 6, 70, 2, 2, 40, 64, True, lengths=rng.integers(0, 41, 70)).check()
    Case(hip, 7, 64, 1, 1, 33, 64, False, lengths=rng.integers(0, 34, 64)).check()


def test_sequences_far_into_the_memory(hip):
    """Matrices of 9 GB, and a sequence in their last rows."""
    batch, n, ld, dim = 70, 8000, 8192, 64
    rows, m = batch * n, 200
    rng = np.random.default_rng(12)
    wide = inputs.to_bf16(rng.normal(size=(m, ld)).astype(np.float32))
    big = [hip.DeviceBuffer(rows * ld * 2) for _ in range(2)]
    d_lse, d_lengths = hip.DeviceBuffer(batch * 2 * n * 4), hip.DeviceBuffer.from_array(np.array([0] * (batch - 1) + [m], np.int32))
    last = (rows - n) * ld * 2
    big[0].upload(wide, last)
    plan = hip.AttentionTraining(batch, 2, n, dim, dim**-0.5, causal=True, kv_heads=1, lengths=d_lengths)
    q, out = big[0], big[1]
    k, v, g, dq, dk, dv = q.at(2 * 128), q.at(2 * 192), q.at(2 * 256), out.at(2 * 128), out.at(2 * 256), out.at(2 * 320)
    hip.attention_training_bf16_dev(plan, q, ld, k, v, ld, out, ld, d_lse)
    hip.attention_backward_bf16_dev(plan, q, ld, k, v, ld, out, ld, d_lse, g, ld, dq, ld, dk, dv, ld)
    hip.device_synchronize()
    got = np.empty((m, ld), np.uint16)
    hip._check(hip._lib.load().st_hip_memcpy_d2h(got.ctypes.data, out.at(last), got.nbytes, None))
    part = lambda x, first, heads: inputs.from_bf16(np.ascontiguousarray(x[:, first:first + heads * dim])).astype(np.float64).reshape(1, m, heads, dim)
    want = plain.training(part(wide, 0, 2), part(wide, 128, 1), part(wide, 192, 1), part(wide, 256, 2), float(np.float32(dim**-0.5)), True, None)
    for name, first, heads in (("out", 0, 2), ("dq", 128, 2), ("dk", 256, 1), ("dv", 320, 1)):
        plain.check(part(got, first, heads), want[name], name)


def test_a_training_step_captured_and_replayed(hip):
    """Attention, the loss over what it gives as logits, and both backward passes, recorded once on a stream without scratch memory and replayed with other
    operands, with eager work and larger calls between the replays."""
    generator = torch.Generator(device="cuda").manual_seed(3)
    batch, heads, kv_heads, n, dim, vocab = 3, 4, 2, 130, 64, 256
    rows, width, fused = batch * n, heads * dim, (heads + 2 * kv_heads) * dim
    bf16 = lambda *shape: torch.randn(*shape, generator=generator, device="cuda").to(torch.bfloat16)
    qkv, table = bf16(rows, fused), torch.randn(8, heads, generator=generator, device="cuda")
    lengths = torch.tensor([130, 0, 71], dtype=torch.int32, device="cuda")
    tokens = torch.randint(-1, vocab, (rows,), generator=generator, device="cuda").int()
    weight = torch.full((rows,), -1.0 / rows, device="cuda")
    assert width == vocab
    out, g, gqkv = bf16(rows, width), bf16(rows, width), bf16(rows, fused)
    lse, gtable = torch.empty(batch, heads, n, device="cuda"), torch.empty(8, heads, device="cuda")
    log_probs, entropies, normalizers = (torch.empty(rows, device="cuda") for _ in range(3))
    ids, top = torch.empty(rows, 3, dtype=torch.int32, device="cuda"), torch.empty(rows, 3, device="cuda")
    plan = hip.AttentionTraining(batch, heads, n, dim, 0.125, causal=True, kv_heads=kv_heads, lengths=lengths.data_ptr(),
                                 position_bias=hip.PositionBias(8, 20, table.data_ptr()))
    q, k, v = qkv.data_ptr(), qkv.data_ptr() + 2 * width, qkv.data_ptr() + 2 * (width + kv_heads * dim)
    gq, gk, gv = gqkv.data_ptr(), gqkv.data_ptr() + 2 * width, gqkv.data_ptr() + 2 * (width + kv_heads * dim)

    def step(stream):
        hip.attention_training_bf16_dev(plan, q, fused, k, v, fused, out.data_ptr(), width, lse.data_ptr(), stream=stream)
        hip.token_log_probs_bf16_dev(rows, vocab, out.data_ptr(), width, tokens.data_ptr(), log_probs.data_ptr(), entropies.data_ptr(),
                                     normalizers.data_ptr(), 3, ids.data_ptr(), top.data_ptr(), stream=stream)
        hip.token_log_probs_backward_bf16_dev(rows, vocab, out.data_ptr(), width, tokens.data_ptr(), normalizers.data_ptr(), entropies.data_ptr(),
                                              weight.data_ptr(), weight.data_ptr(), g.data_ptr(), width, stream=stream)
        hip.attention_backward_bf16_dev(plan, q, fused, k, v, fused, out.data_ptr(), width, lse.data_ptr(), g.data_ptr(), width, gq, fused, gk, gv,
                                        fused, gtable.data_ptr(), stream=stream)

    results = (out, lse, log_probs, entropies, normalizers, ids, top, g, gqkv, gtable)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step(torch.cuda.current_stream().cuda_stream)
    larger = Case(hip, 1, 2, 4, 2, 600, 64, True, buckets=8, far=20)
    try:
        for replay in range(4):
            qkv.mul_(-0.5)
            tokens.add_(1).remainder_(vocab)
            lengths.sub_(1).clamp_(min=0)
            step(None)
            torch.cuda.synchronize()
            want = [x.clone() for x in results]
            for x in results:
                x.fill_(7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(results, want):
                assert torch.equal(x, y), replay
            larger.forward(stream.cuda_stream)
            larger.backward(stream.cuda_stream)  # grows the stream's scratch
            torch.cuda.synchronize()
    finally:
        del graph
        hip.release_scratch(stream.cuda_stream)
        hip.release_scratch(None)


def test_two_threads_on_streams_of_their_own(hip):
    import threading

    cases = [Case(hip, 20 + i, 2, 4, 1, 600, 64, True, buckets=8, far=20) for i in range(2)]
    for case in cases:
        case.forward()
        case.backward()
    want = [case.results() for case in cases]
    failed = []

    def work(i):
        try:
            stream = hip.Stream()
            for _ in range(20):
                cases[i].forward(stream)
                cases[i].backward(stream)
            stream.synchronize()
            stream.destroy()
        except Exception as err:  # reported below
            failed.append(err)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed, failed
    for case, first in zip(cases, want):
        for name, value in case.results().items():
            assert (value == first[name]).all(), name


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,n,lengths,buckets", [(3, 3, 1, None, 0), (4, 2, 1, None, 8), (2, 1, 1500, [1, 1, 0], 0), (2, 2, 40, [1, 0, 1], 8)])
def test_a_single_key_has_all_of_its_row(hip, heads, kv_heads, n, lengths, buckets, causal, dim):
    """Its weight is 1 whatever the score, and the gradients of queries, keys and biases exactly 0."""
    case = Case(hip, 31, 3, heads, kv_heads, n, dim, causal, lengths, buckets=buckets, far=20 if buckets else 0)
    case.check()
    got = case.results()
    for name in got.keys() - {"out", "lse", "dv"}:
        assert (got[name] == 0).all(), name
