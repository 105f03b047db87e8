"""The oracle of trained attention itself: its gradients against differences, and its buckets against the formula."""
import math

import numpy as np
import pytest

import training_oracle as plain


def test_gradients_against_differences():
    """Of sum(out * g), in 64 bits, for the table and for one value each of q, k and v: the formulas themselves."""
    rng = np.random.default_rng(1)
    n, d = 9, 64
    q, k, v, g = (rng.normal(size=(1, n, 2, d)) for _ in range(4))
    k, v = k[:, :, :1], v[:, :, :1]
    table = rng.normal(size=(8, 2))
    value = lambda: (plain.training(q, k, v, g, 0.125, True, None, table, 5, False)["out"][0] * g).sum()
    want = plain.training(q, k, v, g, 0.125, True, None, table, 5, False)
    for name, x, at in (("dq", q, (0, 4, 1, 7)), ("dk", k, (0, 3, 0, 9)), ("dv", v, (0, 2, 0, 1)), ("dtable", table, (2, 1)), ("dtable", table, (5, 0))):
        kept, step = x[at], 1e-5
        x[at] = kept + step
        above = value()
        x[at] = kept - step
        below = value()
        x[at] = kept
        assert abs((above - below) / (2 * step) - want[name][0][at]) < 1e-7, name


@pytest.mark.parametrize("buckets,far,bidirectional", [(32, 128, True), (32, 128, False), (8, 20, False), (64, 300, True), (6, 5, True), (256, 2048, True)])
def test_buckets(buckets, far, bidirectional):
    side = buckets // 2 if bidirectional else buckets
    e = side // 2
    for n in range(-far - 20, far + 21):
        m = abs(n) if bidirectional else max(-n, 0)
        want = m if m < e else min(side - 1, e + math.floor((side - e) * math.log(m / e) / math.log(far / e) + 1e-9))
        assert plain.bucket_of(n, buckets, far, bidirectional) == want + (side if bidirectional and n > 0 else 0), n
