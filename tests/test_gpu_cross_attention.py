"""GPU parity of l3d_cross_attention against softmax in f64 on the same inputs.

Bound, as for the attention over a shared prefix: the probabilities rounded to the
input type (u = 2^-8 bf16, 2^-11 f16, of sum p |v|; f16 below 2^-14 of the row's
largest loses up to 2^-25 each), the f32 scores and exponentials (4e-4 of sum p |v|:
up to 1.4e-4 from the scores, 7.5e-5 twice from the polynomial exponential, the
sums), and the output's rounding (u |o|).  The form for single rows is within it too."""
import math

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _rand(r, shape, dt, dev, std=1.0):
    import torch

    t = torch.from_numpy((std * r.standard_normal(shape)).astype(np.float32)).to(dev)
    return t.to(torch.bfloat16 if dt == "bf16" else torch.float16)


def _ints(v, dev, bits=32):
    import torch

    return torch.tensor(v, dtype=torch.int32 if bits == 32 else torch.int64, device=dev)


def _check(out, q, k, v, rows, keys, dt, scale=None):
    """rows, keys: (first, end) of each sequence."""
    import torch

    Hq, D = q.shape[1:]
    G = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    for b, ((r0, r1), (k0, k1)) in enumerate(zip(rows, keys)):
        if r1 <= r0:
            continue
        if k1 <= k0:
            assert (out[r0:r1] == 0).all(), f"sequence {b} without keys"
            continue
        for h in range(Hq):
            kk, vv = k[k0:k1, h // G].double(), v[k0:k1, h // G].double()
            p = torch.softmax(q[r0:r1, h].double() @ kk.T * scale, -1)
            want, mag = p @ vv, p @ vv.abs()
            bound = mag * (U[dt] + 4e-4) + want.abs() * U[dt] + 1e-6
            if dt == "f16":
                bound = bound + (k1 - k0) * 2.0 ** -25 * vv.abs().amax()
            err = (out[r0:r1, h].double() - want).abs()
            assert (err <= bound).all(), \
                f"sequence {b} head {h}: max err {err.max().item():.3e}, worst ratio {(err / bound).max().item():.2f}"


def _run(ops, dev, rows, keys, Hq, Hkv, D, dt="bf16", layout="packed", equal=False, std=1.0, scale=None, front=0, behind=0):
    """rows, keys: their numbers per sequence; `front` and `behind` rows and keys of no sequence, NaN."""
    import torch

    r = rng(len(rows) * 37 + sum(rows) * 3 + sum(keys) + Hq + D)
    qo, ko = (np.cumsum([0, *n]) + front for n in (rows, keys))
    Tq, Tk = front + sum(rows) + behind, front + sum(keys) + behind
    if layout == "head":  # heads outermost in memory
        q = _rand(r, (Hq, Tq, D), dt, dev, std).transpose(0, 1)
        k, v = (_rand(r, (Hkv, Tk, D), dt, dev, std).transpose(0, 1) for _ in range(2))
    elif layout == "apart":  # normed keys of their own, values inside the projection's rows
        q = _rand(r, (Tq, 2 * Hq, D), dt, dev, std)[:, ::2]
        k, v = _rand(r, (Tk, Hkv, D), dt, dev, std), _rand(r, (Tk, Hkv, 2 * D), dt, dev, std)[..., D:]
    else:
        q = _rand(r, (Tq, Hq, D), dt, dev, std)
        kv = _rand(r, (Tk, Hkv, 2 * D), dt, dev, std)
        k, v = kv[..., :D], kv[..., D:]
    for t in (q, k, v):
        for at in (slice(0, front), slice(t.shape[0] - behind, t.shape[0])):
            t[at] = float("nan")
    out = torch.full((Tq, Hq, D), 7.0, dtype=q.dtype, device=dev)
    bits = 64 if len(rows) % 2 else 32
    got = ops.cross_attention(q, k, v, _ints(ko.tolist(), dev, bits), None if equal else _ints(qo.tolist(), dev, 96 - bits),
                              scale=scale, out=out, check=True)
    assert got is out
    _check(out, q, k, v, list(zip(qo, qo[1:])), list(zip(ko, ko[1:])), dt, scale)
    assert (out[:front] == 7).all() and (out[Tq - behind:] == 7).all()
    return q, k, v, qo, ko, out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,keys,Hq,Hkv,layout", [
    ([1], [1], 1, 1, "packed"),
    ([128], [64], 2, 2, "packed"),
    ([129, 127, 1], [65, 63, 1], 4, 4, "apart"),
    ([5, 0, 300, 70], [77, 10, 0, 200], 8, 2, "packed"),     # a sequence without rows, one without keys
    ([40, 33], [130, 700], 6, 2, "head"),                    # three query heads a key head: 126 rows a tile
    ([300, 20, 1], [257, 1370, 3], 5, 1, "apart"),
    ([700, 1200], [500, 900], 3, 3, "head"),
    ([2049, 100], [1370, 257], 16, 16, "packed"),
])
def test_cross_attention(ops, dev, rows, keys, Hq, Hkv, layout, D, dt):
    _run(ops, dev, rows, keys, Hq, Hkv, D, dt, layout)


@pytest.mark.parametrize("m", [1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 193, 320, 1029])
def test_key_lengths(ops, dev, m):
    _run(ops, dev, [130, 60, 10], [m, m + 1, max(m - 1, 0)], 2, 2, 128)
    _run(ops, dev, [30, 60, 10], [max(m - 1, 0), m, m + 7], 4, 1, 64, front=3, behind=5)


@pytest.mark.parametrize("n", [2, 3, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 385])
def test_row_lengths(ops, dev, n):
    _run(ops, dev, [n, n - 1, n + 1], [100, 257, 30], 4, 2, 64, front=1, behind=2)
    _run(ops, dev, [n] * 3, [100, 257, 30], 4, 4, 128, equal=True)


@pytest.mark.parametrize("N,Hq,Hkv", [(1, 16, 16), (1, 16, 1), (4, 4, 4), (2, 16, 2), (5, 6, 2), (1, 17, 1), (1, 40, 2), (1, 128, 1)])
@pytest.mark.parametrize("dt,D", [("bf16", 64), ("bf16", 128), ("f16", 128)])
def test_few_equal_rows(ops, dev, N, Hq, Hkv, dt, D):
    """Up to 16 rows of a key head take the form for single rows, more the tensor-core one."""
    _run(ops, dev, [N] * 5, [1370, 0, 1, 300, 17], Hq, Hkv, D, dt, "apart", equal=True)


def test_few_equal_rows_behind_others(ops, dev):
    """Keys of no sequence before and behind, through k_offsets; rows in equal groups."""
    import torch

    q, k, v, qo, ko, out = _run(ops, dev, [1] * 4, [100, 7, 0, 64], 4, 2, 64, front=0, equal=True)
    pad = torch.full((3, 2, 64), float("nan"), dtype=k.dtype, device=dev)
    got = ops.cross_attention(q, torch.cat([pad, k, pad]), torch.cat([pad, v, pad]), _ints((ko + 3).tolist(), dev))
    assert torch.equal(got, out)


@pytest.mark.parametrize("B", [31, 32, 33, 200, 1000])
def test_many_sequences(ops, dev, B):
    r = rng(B)
    rows, keys = r.integers(0, 40, B).tolist(), r.integers(0, 150, B).tolist()
    rows[:3], keys[-3:] = [0] * 3, [0] * 3
    _run(ops, dev, rows, keys, 2, 1, 64, layout="head")


@pytest.mark.parametrize("empty", ["rows", "keys"])
def test_most_sequences_most_of_them_empty(ops, dev, empty):
    """2^20 sequences x 64 heads, all but the last two without rows, or without keys."""
    import torch

    B, H, D = 1 << 20, 64, 64
    r = rng(5)
    front = 0 if empty == "rows" else 4096  # rows of sequences without keys, one for each 256th
    q, k, v = (_rand(r, (n, H, D), "bf16", dev) for n in (front + 64, 90, 90))
    qo, ko = (torch.zeros(B + 1, dtype=torch.int32, device=dev) for _ in range(2))
    if front:
        qo[:] = (torch.arange(B + 1, device=dev) // 256).clamp_max(front)
    a, b, c = front, front + 30, front + 64
    qo[-3:] = _ints([a, b, c], dev)
    ko[-2:] = _ints([50, 90], dev)
    out = torch.full_like(q, 7.0)
    ops.cross_attention(q, k, v, ko, qo, out=out, check=True)
    _check(out, q, k, v, [(a, b), (b, c)], [(0, 50), (50, 90)], "bf16")
    assert not out[:a].any()


def test_parts_along_the_keys(ops, dev):
    """Few rows, many keys: an item's keys are cut into parts; ragged, so that some parts are empty."""
    for D in (64, 128):
        _run(ops, dev, [70, 3], [9000, 200], 2, 2, D, front=2, behind=2)
        _run(ops, dev, [20, 20, 20], [4097, 0, 65], 4, 4, D, "f16", equal=True)


def test_scenes_attend_to_themselves(ops, dev):
    import torch

    q, k, v, qo, ko, out = _run(ops, dev, [1500, 700, 90], [1500, 700, 90], 2, 2, 128)
    o = _ints(qo.tolist(), dev)
    assert torch.equal(ops.cross_attention(q, k, v, o, o), out)


def test_scores_far_apart(ops, dev):
    _run(ops, dev, [300, 5], [900, 400], 2, 2, 128, std=12.0)
    _run(ops, dev, [300, 5], [900, 400], 4, 2, 64, "f16", std=12.0, scale=0.5)


@pytest.mark.parametrize("N", [1, 150])
@pytest.mark.parametrize("key", [0, 5, 63, 64, 130, 299])
@pytest.mark.parametrize("val", [math.nan, math.inf, -math.inf])
def test_scores_without_a_softmax(ops, dev, N, key, val):
    import torch

    q, k, v, qo, ko, out = _run(ops, dev, [N, N], [300, 300], 4, 2, 64, equal=True)
    q[..., 3] = 1.0
    k[300 + key, 1, 3] = val
    got = ops.cross_attention(q, k, v, _ints(ko.tolist(), dev))
    assert torch.isfinite(got[:N]).all() and torch.isfinite(got[N:, :2]).all()
    if val == -math.inf:
        assert torch.isfinite(got).all()
    else:
        assert torch.isnan(got[N:, 2:]).all()


def test_neighbours_that_are_not_finite(ops, dev):
    """A sequence's keys stand beside another's: what they hold stays there."""
    import torch

    for N in (1, 200):
        q, k, v, qo, ko, out = _run(ops, dev, [N] * 3, [70, 50, 90], 2, 2, 128, equal=True)
        k[70:120], v[70:120] = float("nan"), float("inf")
        got = ops.cross_attention(q, k, v, _ints(ko.tolist(), dev))
        assert torch.equal(got[:N], out[:N]) and torch.equal(got[2 * N:], out[2 * N:])
        assert torch.isnan(got[N:2 * N]).all()


def test_offsets_outside_the_rows(ops, dev):
    """Offsets are clamped to the rows there are; no keys at all give zeros."""
    import torch

    q, k, v, qo, ko, out = _run(ops, dev, [100, 60], [80, 120], 2, 2, 64)
    got = ops.cross_attention(q, k, v, _ints([-5, 80, 10 ** 9], dev), _ints([-3, 100, 10 ** 9], dev))
    assert torch.equal(got, out)
    for n in (1, 80):  # both forms
        z = ops.cross_attention(q[:2 * n], k[:0], v[:0], _ints([0, 0, 0], dev))
        assert (z == 0).all()
        z = ops.cross_attention(q[:2 * n], k, v, _ints([7, 7, 7], dev))
        assert (z == 0).all()


def test_shared_key_head(ops, dev):
    """Keys and values of one head seen by all (stride 0 between heads)."""
    import torch

    r = rng(4)
    q, k, v = (_rand(r, (200, h, 64), "bf16", dev) for h in (4, 1, 1))
    o = _ints([0, 90, 200], dev)
    want = ops.cross_attention(q, k, v, o, o)
    assert torch.equal(ops.cross_attention(q, k.expand(200, 4, 64), v.expand(200, 4, 64), o, o), want)


def test_results_repeat_and_survive_capture(ops, dev):
    import torch

    r = rng(12)
    for N, Hq in ((1, 8), (260, 4)):
        q, kv = _rand(r, (3 * N, Hq, 128), "bf16", dev), _rand(r, (1200, Hq, 256), "bf16", dev)
        k, v = kv[..., :128], kv[..., 128:]
        ko = _ints([0, 500, 500, 1200], dev)
        first = ops.cross_attention(q, k, v, ko)
        assert all(torch.equal(ops.cross_attention(q, k, v, ko), first) for _ in range(5))
        streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
        torch.cuda.synchronize()
        for s in streams:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.cross_attention(q, k, v, ko))
            graphs.append(g)
        for n in ([0, 500, 500, 1200], [3, 4, 1000, 1001]):
            ko.copy_(_ints(n, dev))
            want = ops.cross_attention(q, k, v, ko)
            torch.cuda.synchronize()
            for _ in range(3):
                for s, g in zip(streams, graphs):
                    with torch.cuda.stream(s):
                        g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_keys_past_32_bits(ops, dev):
    import torch

    D, step = 64, 1 << 26  # elements between rows
    store = torch.empty(79 * step + 2 * D, dtype=torch.bfloat16, device=dev)
    k, v = (store.as_strided((80, 1, D), (step, D, 1), i * D) for i in range(2))
    r = rng(8)
    k.copy_(_rand(r, (80, 1, D), "bf16", dev))
    v.copy_(_rand(r, (80, 1, D), "bf16", dev))
    for n in (1, 40):
        q = _rand(r, (2 * n, 2, D), "bf16", dev)
        out = ops.cross_attention(q, k, v, _ints([0, 9, 80], dev), check=True)
        _check(out, q, k, v, [(0, n), (n, 2 * n)], [(0, 9), (9, 80)], "bf16")


def test_no_room_for_the_workspace(pkg, ops, dev):
    """An allocation that fails is an error, and holds no output."""
    import ctypes
    import sys

    import torch

    q, k = (torch.zeros((n, 2, 64), dtype=torch.bfloat16, device=dev) for n in (4, 9))
    pages, out = k.view(1, 9, 2, 64), torch.zeros_like(q)
    ko, table, n = _ints([0, 9], dev), torch.zeros((4, 1), dtype=torch.int32, device=dev), _ints([9] * 4, dev)
    huge = ctypes.CFUNCTYPE(ctypes.c_size_t)(lambda: 1 << 60)
    size = ctypes.cast(huge, ctypes.c_void_p).value
    before = sys.getrefcount(out)
    for name, args in (("l3d_cross_attention", (q, k, k, ko, None, out)),
                       ("l3d_paged_attention", (q, pages, pages, table, n, out))):
        with pytest.raises(RuntimeError, match="memory"):
            pkg._lib.invoke(name, size, 0, 0.125, *args)
    del args  # (it holds the output too)
    assert sys.getrefcount(out) == before
