"""Attention that is trained, in bf16: its forward and its backward pass against the formulas in 64 bits."""
import numpy as np
import pytest

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
