"""GPU: values that are not finite, of keys that rows see: 0 < p, so p V is infinite with V."""
import math

import pytest

from conftest import rng
from test_gpu_paged import _ints, _rand, _run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("val", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("key", [0, 3, 130, 199])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,dt", [(64, "bf16"), (128, "bf16"), (64, "f16"), (128, "f16")])
def test_values_that_are_not_finite(ops, dev, D, dt, wide, key, val):
    """An infinite V makes what it is weighed into infinite, wherever its key lies; +inf and -inf, or NaN, NaN."""
    import torch

    for N in (1, 4):
        q, kp, vp, table, out = _run_attention(ops, dev, [200, 1, 200], N, 8, 2, D, 16, dt, wide=wide)
        lens = _ints([200, 1, 200], dev)
        at = int(table[0, key // 16]), key % 16
        vp[at][0, 5] = val
        vp[at][1, 7] = val
        vp[int(table[0, 5]), 9, 1, 7] = -math.inf  # key 89
        vp[int(table[1, 0]), 0, :, 0] = val        # a request of one key: a probability of 1
        got = ops.paged_attention(q, kp, vp, table, lens)
        want = out.clone()
        for i in range(N):
            if key < 200 - N + 1 + i:
                want[0, i, :4, 5] = val
                want[0, i, 4:, 7] = val if val == -math.inf else math.nan
            else:
                want[0, i, 4:, 7] = -math.inf
        want[1, N - 1, :, 0] = val
        assert torch.equal(torch.nan_to_num(got, nan=7e3, posinf=8e3, neginf=9e3), torch.nan_to_num(want, nan=7e3, posinf=8e3, neginf=9e3))


@pytest.mark.parametrize("val", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("N", [1, 3, 140])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_packed_values_that_are_not_finite(ops, dev, dt, N, val):
    """The same for packed sequences, in the form for few rows and in the one for many."""
    import torch

    for D in (64, 128):
        r = rng(N + D)
        q = _rand(r, (3 * N, 4, D), dt, dev)
        k, v = (_rand(r, (500, 2, D), dt, dev) for _ in range(2))
        ko = _ints([0, 300, 301, 500], dev)
        want = ops.cross_attention(q, k, v, ko)
        for key in (0, 5, 63, 64, 200, 299):
            v2, w2 = v.clone(), want.clone()
            v2[key, 1, 9], w2[:N, 2:, 9] = val, val
            v2[300, 0, 3], w2[N:2 * N, :2, 3] = val, val
            got = ops.cross_attention(q, k, v2, ko)
            assert torch.equal(torch.nan_to_num(got, nan=7e3, posinf=8e3, neginf=9e3), torch.nan_to_num(w2, nan=7e3, posinf=8e3, neginf=9e3))
