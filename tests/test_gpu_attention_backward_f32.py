"""The backward pass of the f32 attention and of its additive biases against the formulas in 64 bits."""
import numpy as np
import pytest

import training_oracle as plain

pytestmark = pytest.mark.gpu


def wanted(q, k, v, g, scale, causal, z, bias):
    """(contexts, n, d) arrays: {name: (value, bound)} with bounds for f32 throughout."""
    contexts, n, _ = q.shape
    seen = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
    r = {name: ([], []) for name in ("out", "dq", "dk", "dv", "dz", "dbias")}
    for c in range(contexts):
        b = (0.0 if z is None else z[c][None]) + (0.0 if bias is None else bias[c])
        one = plain.head(q[c], k[c], v[c], g[c], scale, seen, b, 0.0)
        ds, e_ds = one["ds"]
        one["dbias"] = one["ds"]
        one["dz"] = ds.sum(0), (e_ds + n * plain.F * np.abs(ds)).sum(0)
        for name in r:
            value, bound = one[name]
            r[name][0].append(value)
            r[name][1].append(bound + 2 * plain.F * np.abs(value) + 2.0**-140)
    return {name: (np.stack(a), np.stack(b)) for name, (a, b) in r.items()}


class Case:
    def __init__(self, hip, seed, contexts, n, d, causal=False, z=False, bias=False, scale=None, spread=1.0, offset=0):
        rng = np.random.default_rng(seed)
        self.hip, self.sizes, self.causal, self.scale = hip, (contexts, n, d), causal, float(np.float32(max(d, 1)**-0.5 if scale is None else scale))
        make = lambda *shape: (spread * rng.normal(size=shape)).astype(np.float32)
        self.x = {name: make(contexts, n, d) for name in ("q", "k", "v", "g")}
        self.x["z"], self.x["bias"] = make(contexts, n) if z else None, make(contexts, n, n) if bias else None
        self.offset = offset  # values before each buffer's first

    def run(self, stream=None):
        x, (contexts, n, d) = self.x, self.sizes
        f64 = {name: None if a is None else a.astype(np.float64) for name, a in x.items()}
        self.want = wanted(f64["q"], f64["k"], f64["v"], f64["g"], self.scale, self.causal, f64["z"], f64["bias"])
        x["out"] = self.want["out"][0].astype(np.float32)
        pad = lambda a: np.concatenate([np.full(self.offset, 7, np.float32), a.ravel(), np.full(5, 7, np.float32)])
        dev = {name: None if a is None else self.hip.DeviceBuffer.from_array(pad(a)) for name, a in x.items()}
        at = lambda name: None if dev[name] is None else dev[name].at(4 * self.offset)
        shapes = {"dq": (contexts, n, d), "dk": (contexts, n, d), "dv": (contexts, n, d)}
        if x["z"] is not None:
            shapes["dz"] = (contexts, n)
        if x["bias"] is not None:
            shapes["dbias"] = (contexts, n, n)
        out = {name: self.hip.DeviceBuffer.from_array(pad(np.full(shape, 7, np.float32))) for name, shape in shapes.items()}
        to = lambda name: out[name].at(4 * self.offset) if name in out else None
        self.hip.attention_backward_f32_dev(contexts, n, d, self.scale, self.causal, at("q"), at("k"), at("v"), at("z"), at("bias"), at("out"), at("g"),
                                            to("dq"), to("dk"), to("dv"), to("dz"), to("dbias"), stream=stream)
        self.hip.device_synchronize()
        got = {}
        for name, shape in shapes.items():
            size = int(np.prod(shape))
            flat = out[name].to_array(np.float32, self.offset + size + 5)
            assert (flat[:self.offset] == 7).all() and (flat[self.offset + size:] == 7).all(), f"{name}: values beside"
            got[name] = flat[self.offset:self.offset + size].reshape(shape)
        return got

    def check(self, what=""):
        got = self.run()
        for name in got:
            plain.check(got[name], self.want[name], f"{what} {name}")
        return got


CASES = [(1, 1, 1), (2, 7, 3), (3, 33, 8), (2, 19, 5), (1, 40, 16), (4, 64, 64), (2, 129, 64), (3, 200, 32), (1, 130, 80), (2, 96, 256), (1, 70, 200), (5, 128, 96),
         (8, 31, 33), (1, 300, 128), (2, 2, 100), (1, 161, 130)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("z,bias", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("contexts,n,d", CASES)
def test_sizes(hip, contexts, n, d, causal, z, bias):
    Case(hip, contexts + n + d, contexts, n, d, causal, z, bias).check()


@pytest.mark.parametrize("offset", [1, 2, 3, 4])
@pytest.mark.parametrize("n,d", [(64, 64), (50, 24), (61, 20)])
def test_buffers_at_any_boundary(hip, n, d, offset):
    Case(hip, offset, 2, n, d, True, True, True, offset=offset).check()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(hip, scale):
    Case(hip, 1, 2, 75, 32, False, True, True, scale=scale).check()


def test_sharp_rows(hip):
    Case(hip, 2, 2, 90, 64, False, False, True, spread=5.0).check()


def test_keys_barred_by_minus_infinity(hip):
    """Biases of -infinity bar pairs, whole keys and whole rows."""
    for causal in (False, True):
        case = Case(hip, 3, 2, 70, 64, causal, True, True)
        case.x["bias"][0, 5, ::3] = -np.inf
        case.x["bias"][1, 9] = -np.inf  # a row with nothing
        case.x["z"][0, 20:40] = -np.inf
        got = case.check(f"causal {causal}")
        assert (got["dq"][1, 9] == 0).all() and (got["dbias"][1, 9] == 0).all() and (got["dk"][0, 20:40] == 0).all()
        assert (got["dz"][0, 20:40] == 0).all() and (got["dv"][0, 20:40] == 0).all()


def test_biases_of_heads_without_values(hip):
    case = Case(hip, 4, 2, 40, 0, False, True, True)
    got = case.run()
    assert (got["dz"] == 0).all() and (got["dbias"] == 0).all()


@pytest.mark.parametrize("causal", [False, True])
def test_behind_the_forward_pass_of_tensors(hip, causal):
    """Tensor.scaled_dot_attention and its gradients, as a training step calls them, against differences of the loss in 64 bits."""
    from spiraltorch_amd import Tensor

    rng = np.random.default_rng(7)
    contexts, n, d, scale = 3, 45, 24, 0.2
    shapes = {"q": (contexts * n, d), "k": (contexts * n, d), "v": (contexts * n, d), "z": (contexts, n), "bias": (contexts * n, n)}
    x = {name: rng.normal(size=shape).astype(np.float32) for name, shape in shapes.items()}
    g = rng.normal(size=(contexts * n, d)).astype(np.float32)
    t = {name: Tensor.from_numpy(a) for name, a in x.items()}
    kept = dict(contexts=contexts, sequence=n, scale=scale, z_bias=t["z"], attn_bias=t["bias"], causal=causal)
    out = t["q"].scaled_dot_attention(t["k"], t["v"], **kept)
    gradients = t["q"].scaled_dot_attention_backward(t["k"], t["v"], out, Tensor.from_numpy(g), **kept)

    def loss(x):
        q, k, v = (x[name].reshape(contexts, n, d) for name in ("q", "k", "v"))
        s = scale * q @ k.transpose(0, 2, 1) + x["z"][:, None] + x["bias"].reshape(contexts, n, n)
        if causal:
            s = np.where(np.tril(np.ones((n, n), bool)), s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        return ((p / p.sum(-1, keepdims=True)) @ v * g.reshape(contexts, n, d)).sum()

    x = {name: a.astype(np.float64) for name, a in x.items()}
    for name, gradient in zip(shapes, gradients):
        for _ in range(5):
            at, step = tuple(int(rng.integers(0, m)) for m in shapes[name]), 1e-5
            value = x[name][at]
            x[name][at] = value + step
            above = loss(x)
            x[name][at] = value - step
            below = loss(x)
            x[name][at] = value
            # the difference's own error is about step^2 and 1e-16 / step; the gradient's is f32's
            assert abs((above - below) / (2 * step) - gradient.numpy()[at]) < 2e-5, (name, at)


def test_tensor_gradients_that_are_refused(hip):
    from spiraltorch_amd import Tensor, TensorError

    t, other = Tensor.zeros(6, 4), Tensor.zeros(6, 5)
    for args, kw in (((t, t, t, other), {}), ((t, other, t, t), {}), ((t, t, t, t), {"z_bias": Tensor.zeros(3, 2)}), ((t, t, t, t), {"attn_bias": t}),
                     ((t, t, t, t), {"scale": float("nan")}), ((t, t, t, Tensor(6, 4, [float("inf")] * 24)), {})):
        with pytest.raises(TensorError):
            t.scaled_dot_attention_backward(*args, **{"contexts": 2, "sequence": 3, "scale": 1.0, **kw})
    assert t.scaled_dot_attention_backward(t, t, t, t, contexts=2, sequence=3, scale=1.0)[3:] == (None, None)
    empty = Tensor.zeros(0, 4)
    assert empty.scaled_dot_attention_backward(empty, empty, empty, empty, contexts=0, sequence=3, scale=1.0)[0].shape() == (0, 4)
