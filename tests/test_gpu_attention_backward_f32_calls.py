"""The f32 attention's backward pass in many contexts at once, again, captured and from two threads."""
import threading

import numpy as np
import pytest
import torch

import training_oracle as plain
from test_gpu_attention_backward_f32 import wanted

pytestmark = pytest.mark.gpu


class Buffers:
    """A call's operands and results in torch's memory; `out` is what 64 bits give, where a check needs it, or any values."""

    def __init__(self, seed, contexts, n, d, causal, biased):
        generator = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *shape: torch.randn(*shape, generator=generator, device="cuda")
        self.sizes, self.causal, self.scale = (contexts, n, d), causal, float(np.float32(d**-0.5))
        self.x = {name: make(contexts, n, d) for name in ("q", "k", "v", "out", "g")}
        self.x.update(z=make(contexts, n) if biased else None, bias=make(contexts, n, n) if biased else None)
        self.y = {"d" + name: torch.empty_like(self.x[name]) for name in ("q", "k", "v")}
        if biased:
            self.y.update(dz=torch.empty(contexts, n, device="cuda"), dbias=torch.empty(contexts, n, n, device="cuda"))
        torch.cuda.synchronize()

    def part(self, first, last):
        """The same operands of some of the contexts, with results of its own."""
        other = object.__new__(Buffers)
        other.sizes, other.causal, other.scale = (last - first, *self.sizes[1:]), self.causal, self.scale
        cut = lambda a: None if a is None else a[first:last].clone()
        other.x, other.y = {name: cut(a) for name, a in self.x.items()}, {name: torch.empty_like(a[first:last]) for name, a in self.y.items()}
        torch.cuda.synchronize()
        return other

    def run(self, hip, stream=None):
        at = lambda a: None if a is None else a.data_ptr()
        x, y = self.x, self.y
        hip.attention_backward_f32_dev(*self.sizes, self.scale, self.causal, *(at(x[name]) for name in ("q", "k", "v", "z", "bias", "out", "g")),
                                       *(at(y.get(name)) for name in ("dq", "dk", "dv", "dz", "dbias")), stream=stream)

    def results(self):
        torch.cuda.synchronize()
        return {name: a.clone() for name, a in self.y.items()}

    def want(self, contexts):
        f64 = {name: None if a is None else a[contexts].cpu().numpy().astype(np.float64) for name, a in self.x.items()}
        return wanted(f64["q"], f64["k"], f64["v"], f64["g"], self.scale, self.causal, f64["z"], f64["bias"])


@pytest.mark.parametrize("n,d,contexts", [(1024, 32, 65), (1000, 64, 70), (1024, 72, 65), (1024, 96, 65), (1011, 90, 66), (1024, 128, 65), (1000, 200, 70)])
@pytest.mark.parametrize("causal", [False, True])
def test_more_pairs_than_are_kept(hip, n, d, contexts, causal):
    """Above 2^26 pairs dq works ds out again."""
    assert contexts * n * n > 1 << 26
    case, some = Buffers(n + d, contexts, n, d, causal, False), [0, contexts - 1]
    want = case.want(some)
    case.x["out"][some] = torch.from_numpy(want["out"][0].astype(np.float32)).cuda()
    torch.cuda.synchronize()
    case.run(hip)
    for name, a in case.results().items():
        plain.check(a[some].cpu().numpy(), want[name], name)


@pytest.mark.parametrize("n,d,contexts", [(40, 80, 500), (64, 96, 1100), (33, 128, 400), (64, 65, 1025)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_many_contexts(hip, n, d, contexts, causal, biased):
    """Enough of them for workgroups of two wavefronts."""
    case, some = Buffers(n + d, contexts, n, d, causal, biased), [0, 7, contexts // 2, contexts - 1]
    want = case.want(some)
    case.x["out"][some] = torch.from_numpy(want["out"][0].astype(np.float32)).cuda()
    torch.cuda.synchronize()
    case.run(hip)
    for name, a in case.results().items():
        plain.check(a[some].cpu().numpy(), want[name], name)


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n,d", [(150, 64), (130, 80), (70, 256), (61, 31)])
def test_the_same_bits_again_and_in_fewer_contexts(hip, n, d, biased):
    case = Buffers(1, 12, n, d, True, biased)
    case.run(hip)
    first = case.results()
    for a in case.y.values():
        a.fill_(7)
    torch.cuda.synchronize()
    case.run(hip)
    again = case.results()
    few = case.part(3, 8)
    few.run(hip)
    few = few.results()
    for name, a in first.items():
        assert torch.equal(a, again[name]), name
        assert torch.equal(a[3:8], few[name]), name


@pytest.mark.parametrize("biased", [False, True])
def test_captured_and_replayed(hip, biased):
    """Recorded on a stream without scratch memory, replayed with other operands, larger calls between the replays."""
    case, larger = Buffers(2, 5, 140, 64, True, biased), Buffers(3, 8, 400, 64, False, False)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        case.run(hip, torch.cuda.current_stream().cuda_stream)
    try:
        for replay in range(4):
            for name in ("q", "k", "g"):
                case.x[name].mul_(-0.5)
            torch.cuda.synchronize()
            case.run(hip)
            want = case.results()
            for a in case.y.values():
                a.fill_(7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            for name, a in case.results().items():
                assert torch.equal(a, want[name]), (replay, name)
            larger.run(hip, stream.cuda_stream)  # grows the stream's scratch
            torch.cuda.synchronize()
    finally:
        del graph
        hip.release_scratch(stream.cuda_stream)
        hip.release_scratch(None)


def test_two_threads_on_streams_of_their_own(hip):
    cases = [Buffers(10 + i, 6, 200, 48, True, False) for i in range(2)]
    for case in cases:
        case.run(hip)
    want = [case.results() for case in cases]
    failed = []

    def work(i):
        try:
            stream = hip.Stream()
            for _ in range(20):
                cases[i].run(hip, stream)
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
        for name, a in case.results().items():
            assert torch.equal(a, first[name]), name


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("d", [1, 64, 80, 200])
def test_a_single_key_has_all_of_every_row(hip, d, biased, causal):
    """Its weight is 1 whatever the scores, and everything but dv exactly 0."""
    case = Buffers(d, 37, 1, d, causal, biased)
    case.x["out"].copy_(case.x["v"])
    case.run(hip)
    got = case.results()
    for name in got.keys() - {"dv"}:
        assert (got[name] == 0).all(), name
    # p = 2^(s - lse) with lse = s + log2(1), s below 16 rounded twice (to 2^-21 each at the most) in units of log2 e: off by less than 2^-20, and rounded
    s = (case.x["q"] * case.x["k"]).sum((1, 2)) * case.scale + (case.x["z"][:, 0] + case.x["bias"][:, 0, 0] if biased else 0)
    assert s.abs().max() * 1.4427 < 15.9
    assert ((got["dv"] - case.x["g"]).abs() <= 2.0**-20 * case.x["g"].abs()).all()


PARTS = [(1, 1000, 64), (2, 700, 80), (1, 1024, 128), (1, 530, 256), (3, 401, 200), (1, 1500, 8), (2, 999, 31), (1, 2048, 96)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("contexts,n,d", PARTS)
def test_few_long_contexts(hip, contexts, n, d, biased, causal):
    """Several workgroups to a tile, whose sums are added up behind them; keys that biases bar, and a row that sees nothing."""
    case = Buffers(n + d, contexts, n, d, causal, biased)
    if biased:
        case.x["z"][0, n // 3:n // 2] = -torch.inf
        case.x["bias"][0, n - 5] = -torch.inf
        case.x["bias"][contexts - 1, 40, ::2] = -torch.inf
    want = case.want(list(range(contexts)))
    case.x["out"].copy_(torch.from_numpy(want["out"][0].astype(np.float32)))
    torch.cuda.synchronize()
    case.run(hip)
    first = case.results()
    for name, a in first.items():
        plain.check(a.cpu().numpy(), want[name], name)
    for a in case.y.values():
        a.fill_(7)
    torch.cuda.synchronize()
    case.run(hip)
    for name, a in case.results().items():
        assert torch.equal(a, first[name]), name


def test_few_long_contexts_captured_and_replayed(hip):
    case, larger = Buffers(21, 1, 1100, 64, True, True), Buffers(22, 1, 2000, 96, False, False)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        case.run(hip, torch.cuda.current_stream().cuda_stream)
    try:
        for replay in range(3):
            case.x["q"].mul_(-0.5)
            torch.cuda.synchronize()
            case.run(hip)
            want = case.results()
            for a in case.y.values():
                a.fill_(7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            for name, a in case.results().items():
                assert torch.equal(a, want[name]), (replay, name)
            larger.run(hip, stream.cuda_stream)  # grows the stream's scratch
            torch.cuda.synchronize()
    finally:
        del graph
        hip.release_scratch(stream.cuda_stream)
        hip.release_scratch(None)
