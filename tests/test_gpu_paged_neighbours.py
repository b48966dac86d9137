"""GPU: what a key of no weight, a bad page or a bad length does to the rest, held to the bounds of test_gpu_paged and
test_gpu_cross_attention."""
import math

import pytest

from conftest import rng
from test_gpu_cross_attention import _check
from test_gpu_paged import _check_attention, _ints, _rand, _run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("key", [0, 7, 100, 199])
@pytest.mark.parametrize("wide", [False, True])
def test_a_score_of_minus_infinity_has_no_weight(ops, dev, key, wide):
    import torch

    for dt in ("bf16", "f16"):
        q, kp, vp, table, _ = _run_attention(ops, dev, [200, 200], 2, 4, 2, 128, 16, dt, wide=wide)
        q[..., 3] = 1.0
        kp[int(table[1, key // 16]), key % 16, 1, 3] = -math.inf
        got = ops.paged_attention(q, kp, vp, table, _ints([200, 200], dev))
        _check_attention(got, q, kp, vp, table, [200, 200], dt)


@pytest.mark.parametrize("N", [1, 150])
@pytest.mark.parametrize("key", [0, 63, 64, 299])
def test_a_packed_score_of_minus_infinity_has_no_weight(ops, dev, N, key):
    r = rng(key)
    for dt in ("bf16", "f16"):
        q, k, v = (_rand(r, s, dt, dev) for s in ((2 * N, 4, 64), (600, 2, 64), (600, 2, 64)))
        q[..., 3] = 1.0
        k[300 + key, 1, 3] = -math.inf
        got = ops.cross_attention(q, k, v, _ints([0, 300, 600], dev))
        _check(got, q, k, v, [(0, N), (N, 2 * N)], [(0, 300), (300, 600)], dt)


@pytest.mark.parametrize("wide", [False, True])
def test_beside_a_bad_page_or_length(ops, dev, wide):
    """The requests beside one that comes out NaN are as near as ever."""
    import torch

    for D in (64, 128):
        lens = [300, 280, 260, 40]
        q, kp, vp, table, out = _run_attention(ops, dev, lens, 1, 8, 2, D, 16, wide=wide)
        tab = table.clone()
        tab[0, 7] = kp.shape[0]
        got = ops.paged_attention(q, kp, vp, tab, _ints([300, 280, 10 ** 9, 40], dev))
        assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all()
        for b in (1, 3):
            _check_attention(got[b:b + 1], q[b:b + 1], kp, vp, table[b:b + 1], [lens[b]], "bf16")
