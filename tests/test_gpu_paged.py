"""GPU parity of the paged cache: l3d_paged_append and l3d_paged_attention against
their definitions in f64 on the same inputs.

Bounds.  u is half a step of the type (2^-8 bf16, 2^-11 f16).
append: u |y| for the output's rounding; 2e-6 (|lo| + |hi|) of the pair for the f32
norm (128 squares added as a tree: 2e-7; square root, division, two products: 3e-7)
and the rotation (angle to 2^-25 of a turn, 2e-7 rad; sine and cosine to 2 ulp, two
products and a sum: 4e-7); f16 steps below 2^-14: 2^-25.
attention: u |o| for the output; of sum p |v|: 1.4e-4 for the scores (an f32 sum of
128 products is off by at most 128 2^-24 |q| |k| scale, about 7e-5 at |q| |k| = 100;
counted in the sum over and under the fraction), 2^-16 for the two parts of a
probability and 1e-5 for the sums; f16 parts below 2^-14: 2^-25 |v| a key."""
import math

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _dt(dt):
    import torch

    return torch.bfloat16 if dt == "bf16" else torch.float16


def _rand(r, shape, dt, dev, std=1.0, mean=0.0):
    import torch

    return torch.from_numpy((mean + std * r.standard_normal(shape)).astype(np.float32)).to(dev).to(_dt(dt))


def _ints(v, dev, bits=32):
    import torch

    return torch.tensor(v, dtype=torch.int32 if bits == 32 else torch.int64, device=dev)


def _pages(r, counts, size, H, D, dt, dev, layout="token", fill=None):
    """A cache whose pages lie scattered, and the table for `counts` tokens of each request."""
    import torch

    need = [-(-n // size) for n in counts]
    total = sum(need) + 2
    shape = {"token": (total, size, H, D), "head": (total, H, size, D), "both": (total, 2, size, H, D)}[layout]

    def one(shape):
        return _rand(r, shape, dt, dev) if fill is None else torch.full(shape, fill, dtype=_dt(dt), device=dev)
    if layout == "both":  # keys and values of a page side by side
        kv = one(shape)
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = one(shape), one(shape)
        if layout == "head":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = r.permutation(total)
    table, at = np.full((len(need), max(max(need), 1)), -1, np.int64), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return k, v, _ints(table.tolist(), dev), order[at:]


# ------------------------------------------------------------------- append
def _rows(table, size, b, place):
    return int(table[b, place // size]), place % size


def _turned(x, w, rope, pos, eps):
    """Norm and rotation of x [n, H, D] at pos [n, axes], in f64; and |lo| + |hi| of each element's pair."""
    import torch

    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    y, mag = x.clone(), x.abs()
    if rope is not None:
        f, ax, pairs, h = rope.want, rope.axis.tolist(), len(rope.want), rope.half
        for i in range(pairs):
            lo, hi = (2 * i, 2 * i + 1) if h == 0 else (i // h * 2 * h + i % h, i // h * 2 * h + i % h + h)
            t = (pos[:, ax[i]].double() * f[i])[:, None]
            y[..., lo] = x[..., lo] * torch.cos(t) - x[..., hi] * torch.sin(t)
            y[..., hi] = x[..., hi] * torch.cos(t) + x[..., lo] * torch.sin(t)
            # The frequency's two f32 parts hold 2 x 24 bits, and the f64 products here and there round at 2^-53: the
            # angle t is off by up to 2^-48 |t| (2^-8 radians at position 2^40, which the 2e-6 of _close does not cover).
            far = 1 + t.abs() * (2.0 ** -48 / 2e-6)
            mag[..., lo] = mag[..., hi] = (x[..., lo].abs() + x[..., hi].abs()) * far
    return y, mag


def _close(got, want, mag, dt, what):
    err = (got.double() - want).abs()
    bound = U[dt] * want.abs() + 2e-6 * mag + 2.0 ** -25
    assert (err <= bound).all(), f"{what}: max err {err.max().item():.3e}, worst ratio {(err / bound).max().item():.2f}"


def _rope(ops, D, sections, layout, theta, dev):
    r = ops.RotaryAxes(D, sections, theta=theta, layout=layout, device=dev)
    r.want = np.concatenate([float(theta) ** (-np.arange(n) / n) for n in sections])
    return r


def _run_append(ops, dev, held, new, Hq, Hkv, D, size, rope=None, positions=None, weights="one", dt="bf16",
                layout="token", bits=32, inplace=False, eps=1e-6, front=0, behind=0):
    import torch

    r = rng(len(held) * 101 + sum(new) * 7 + Hq * 3 + D + size)
    B = len(held)
    T = front + sum(new) + behind
    k_pages, v_pages, table, _ = _pages(r, [a + b for a, b in zip(held, new)], size, Hkv, D, dt, dev, layout)
    qkv = _rand(r, (T, Hq + 2 * Hkv, D), dt, dev, 1.5)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    q0, k0, v0 = q.clone(), k_pages.clone(), v_pages.clone()
    qw = kw = None
    if weights:
        qw = _rand(r, (D,) if weights == "one" else (Hq, D), dt, dev, 0.2, 1.0)
        kw = _rand(r, (D,) if weights == "one" else (Hkv, D), dt, dev, 0.2, 1.0)
        if weights == "one":
            qw = qw.float()  # of another type than x
    equal = len(set(new)) == 1 and not front and not behind
    offsets = None if equal else _ints((np.cumsum([0, *new]) + front).tolist(), dev, bits)
    out = q if inplace else torch.full_like(q0, 7.0)
    pos = None if positions is None else _ints(positions(r, T), dev, bits)
    got = ops.paged_append(q, k, v, k_pages, v_pages, table, _ints(held, dev, bits), offsets, rope, pos, qw, kw, eps, out)
    torch.cuda.synchronize()
    assert got is out
    t = front
    for b in range(B):
        place = torch.arange(held[b], held[b] + new[b], device=dev)
        rows = slice(t, t + new[b])
        p = place[:, None].expand(-1, 8) if pos is None else pos[rows]
        _close(got[rows], *_turned(q0[rows], qw, rope, p, eps), dt, f"q of request {b}")
        page = table[b].long()[place // size]
        _close(k_pages[page, place % size], *_turned(k[rows], kw, rope, p, eps), dt, f"k of request {b}")
        assert torch.equal(v_pages[page, place % size], v[rows])
        k_pages[page, place % size] = k0[page, place % size]
        v_pages[page, place % size] = v0[page, place % size]
        t += new[b]
    assert torch.equal(k_pages, k0) and torch.equal(v_pages, v0)  # nothing else was written
    for rows in (slice(0, front), slice(t, T)):
        assert torch.equal(got[rows], q0[rows] if inplace else torch.full_like(q0[rows], 7.0))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("held,new,Hq,Hkv,size,layout", [
    ([0], [1], 1, 1, 1, "token"),
    ([15, 16, 17, 0], [1, 1, 1, 1], 8, 2, 16, "token"),
    ([5, 0, 31], [3, 0, 40], 4, 4, 16, "head"),
    ([100, 7], [29, 1], 12, 3, 48, "both"),
    ([0, 3, 0, 9, 2], [700, 1, 333, 0, 90], 16, 1, 64, "token"),   # several tokens a block
])
def test_append(ops, dev, held, new, Hq, Hkv, size, layout, D, dt):
    _run_append(ops, dev, held, new, Hq, Hkv, D, size, _rope(ops, D, (D // 2,), "half", 10000.0, dev), dt=dt,
                layout=layout, bits=64 if len(held) % 2 else 32)


@pytest.mark.parametrize("D,sections,rope_layout", [
    (128, (16, 24, 24), "half"), (128, (48,), "interleaved"), (128, (21, 21, 21), "interleaved"), (128, (8, 16), "half"),
    (128, (16, 16, 16), "axis"), (64, (16, 16), "axis"), (64, (5, 3, 7), "interleaved"), (64, (8, 8), "axis"),
    (64, (32,), "half"), (64, (1,), "interleaved"), (64, (3, 5), "half"),
])
@pytest.mark.parametrize("weights", ["one", "head", None])
def test_append_axes(ops, dev, D, sections, rope_layout, weights):
    """Positions on several axes, far ones and negative ones among them."""
    def positions(r, T):
        p = r.integers(-5, 1000, (T, len(sections)))
        p[0, 0], p[-1, -1] = 1 << 30, 131071
        return p.tolist()
    _run_append(ops, dev, [3, 40], [6, 2], 4, 2, D, 16, _rope(ops, D, sections, rope_layout, 10000.0, dev), positions,
                weights, layout="both")


def test_append_far_positions(ops, dev):
    """64-bit positions, whose angle a 32-bit product loses altogether."""
    _run_append(ops, dev, [3], [4], 2, 1, 64, 16, _rope(ops, 64, (32,), "half", 10000.0, dev),
                lambda r, T: [[1 << 33], [(1 << 40) + 1], [-(1 << 33)], [0]], bits=64, dt="f16")


def test_append_without_rotation(ops, dev):
    _run_append(ops, dev, [3, 9], [2, 2], 3, 3, 128, 8, weights="head")
    _run_append(ops, dev, [3, 9], [2, 2], 3, 3, 128, 8, weights=None, dt="f16")


@pytest.mark.parametrize("inplace", [False, True])
def test_append_rows_of_no_request(ops, dev, inplace):
    _run_append(ops, dev, [3, 0, 30], [2, 0, 300], 4, 2, 64, 16, _rope(ops, 64, (32,), "half", 1e6, dev), inplace=inplace,
                front=5, behind=9)


def test_append_eps_and_zero_rows(ops, dev):
    """A head of zeros stays zero, for any eps above it."""
    import torch

    q = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device=dev)
    w = torch.ones(64, device=dev)
    pages = torch.ones(2, 4, 1, 64, dtype=torch.bfloat16, device=dev)
    out = ops.paged_append(q, q, q, pages, pages.clone(), _ints([[0], [1]], dev), _ints([0, 3], dev), q_weight=w, k_weight=w)
    torch.cuda.synchronize()
    assert (out == 0).all() and (pages[0, 0] == 0).all() and (pages[1, 3] == 0).all() and (pages[0, 1:] == 1).all()


def test_append_without_a_place(ops, dev):
    """Tokens past the table or on a page that is none of the cache: not stored, q NaN; the others as ever."""
    import torch

    r = rng(5)
    T, D = 7, 64
    q, k, v = (_rand(r, (T, 2, D), "bf16", dev) for _ in range(3))
    kp, vp = (_rand(r, (4, 8, 2, D), "bf16", dev) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    #          one slot left  bad page   negative page  fine   held negative
    table = _ints([[0, 1], [2, 4], [-1, 3], [3, 2], [2, 2]], dev)
    held = _ints([15, 8, 0, 0, -3], dev)
    out = ops.paged_append(q, k, v, kp, vp, table, held, _ints([0, 3, 4, 5, 6, 7], dev))
    torch.cuda.synchronize()
    nan = torch.isnan(out).all(-1).all(-1).tolist()
    assert nan == [False, True, True, True, True, False, True]
    assert torch.equal(out[0], q[0]) and torch.equal(out[5], q[5])
    k0[1, 7], v0[1, 7], k0[3, 0], v0[3, 0] = k[0], v[0], k[5], v[5]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


# ---------------------------------------------------------------- attention
def _want(q, k, v, n, scale):
    """Rows q [N, Hq, D] over the first n of k and v [.., Hkv, D]; the result and sum p |v|, f64."""
    import torch

    N, Hq, D = q.shape
    G = Hq // k.shape[1]
    k, v = (t[:max(n, 0)].double().repeat_interleave(G, 1) for t in (k, v))
    o, mag = torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device), torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device)
    for i in range(N):
        m = n - N + 1 + i
        if m <= 0:
            continue
        p = torch.softmax(torch.einsum("hd,shd->hs", q[i].double(), k[:m]) * scale, -1)
        o[i], mag[i] = torch.einsum("hs,shd->hd", p, v[:m]), torch.einsum("hs,shd->hd", p, v[:m].abs())
    return o, mag


def _check_attention(out, q, k_pages, v_pages, table, lens, dt, scale=None):
    B, N, Hq, D = q.shape
    size = k_pages.shape[1]
    scale = D ** -0.5 if scale is None else scale
    for b in range(B):
        n = max(lens[b], 0)
        ids = table[b, :-(-n // size)].long()
        k, v = k_pages[ids].flatten(0, 1), v_pages[ids].flatten(0, 1)
        o, mag = _want(q[b], k, v, n, scale)
        bound = U[dt] * o.abs() + (1.4e-4 + 2.0 ** -16 + 1e-5) * mag + 1e-7
        if dt == "f16" and n:
            bound = bound + n * 2.0 ** -25 * v[:n].double().abs().amax() + 2.0 ** -25
        err = (out[b].double() - o).abs()
        assert (err <= bound).all(), \
            f"request {b} of {n} keys: max err {err.max().item():.3e}, worst ratio {(err / bound).max().item():.2f}"


def _run_attention(ops, dev, lens, N, Hq, Hkv, D, size, dt="bf16", layout="token", std=1.0, scale=None, bits=32,
                   wide=False):
    """Slots that no request has reached and pages of nobody hold NaN.  `wide`: tables with room for many more
    keys, which few requests then divide over the device."""
    import torch

    r = rng(len(lens) * 31 + N * 7 + Hq + D + size + sum(lens))
    kp, vp, table, free = _pages(r, lens, size, Hkv, D, dt, dev, layout)
    q = _rand(r, (len(lens), N, Hq, D), dt, dev, std)
    for b, n in enumerate(lens):
        if n > 0 and n % size:
            kp[table[b, n // size].long(), n % size:] = float("nan")
            vp[table[b, n // size].long(), n % size:] = float("inf") if b % 2 else float("nan")
    for p in free.tolist():
        kp[p] = vp[p] = float("nan")
    if wide:
        table = torch.cat([table, torch.full((len(lens), 9000 // size), -1, dtype=torch.int32, device=dev)], 1)
    out = ops.paged_attention(q, kp, vp, table, _ints(lens, dev, bits), scale=scale, check=True)
    _check_attention(out, q, kp, vp, table, lens, dt, scale)
    return q, kp, vp, table, out


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,N,Hq,Hkv,size,layout", [
    ([1], 1, 1, 1, 16, "token"),
    ([300], 1, 8, 2, 16, "token"),
    ([0, 1, 15, 16, 17, 2000, 31, 33, 0], 1, 16, 4, 16, "head"),
    ([257, 64], 1, 4, 4, 1, "token"),
    ([97, 4097, 48], 1, 12, 3, 48, "both"),
    ([70, 3, 1, 0, 900], 4, 6, 3, 16, "token"),     # a few tokens; two requests hold fewer than those
    ([130, 20], 16, 16, 2, 32, "both"),             # 128 rows of a key head
    ([65, 40], 7, 5, 1, 8, "head"),                 # 35 rows
    ([5000] * 40, 1, 8, 8, 64, "token"),
    ([9] * 300, 1, 4, 2, 16, "token"),              # more requests than threads of a block
    ([20000], 2, 16, 2, 256, "token"),
])
def test_paged_attention(ops, dev, lens, N, Hq, Hkv, size, layout, D, dt):
    _run_attention(ops, dev, lens, N, Hq, Hkv, D, size, dt, layout, bits=64 if len(lens) % 2 else 32)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 511, 512, 513, 4095, 4096, 4097])
@pytest.mark.parametrize("wide", [False, True])
def test_paged_lengths(ops, dev, n, wide):
    _run_attention(ops, dev, [n, n + 1, max(n - 1, 0)], 1, 8, 2, 128, 16, wide=wide)
    _run_attention(ops, dev, [n, n + 1, max(n - 1, 0)], 3, 2, 2, 64, 24, wide=wide)
    _run_attention(ops, dev, [n, 0, 1], 5, 4, 2, 64, 1 if n < 600 else 40, "f16", wide=wide)  # ten rows


def test_paged_attention_scores_far_apart(ops, dev):
    """Scores of hundreds: the maximum moves many times, most probabilities vanish."""
    _run_attention(ops, dev, [3000, 700], 1, 8, 2, 128, 16, std=12.0)
    _run_attention(ops, dev, [3000, 700], 2, 8, 2, 64, 16, std=12.0, dt="f16", scale=0.5)


def test_paged_attention_many_requests(ops, dev):
    r = rng(77)
    lens = r.integers(0, 400, 4096).tolist()
    lens[:40], lens[-30:] = [0] * 40, [0] * 30
    _run_attention(ops, dev, lens, 1, 2, 1, 64, 64)


def test_one_row_form_and_strides(ops, dev):
    import torch

    q, kp, vp, table, out = _run_attention(ops, dev, [100, 30], 1, 8, 2, 64, 16)
    lens = _ints([100, 30], dev)
    assert torch.equal(ops.paged_attention(q[:, 0], kp, vp, table, lens), out[:, 0])
    # q inside a projection's rows, out in the middle of a larger tensor, a table with room behind each row
    wide = torch.zeros(2, 1, 20, 64, dtype=q.dtype, device=dev)
    wide[:, :, 3:11] = q
    big = torch.full((2, 3, 8, 64), 5.0, dtype=q.dtype, device=dev)
    tab = torch.full((2, table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device=dev)
    tab[:, 2:2 + table.shape[1]] = table
    ops.paged_attention(wide[:, :, 3:11], kp, vp, tab[:, 2:], lens, out=big[:, 1:2])
    assert torch.equal(big[:, 1:2], out) and (big[:, 0] == 5).all() and (big[:, 2] == 5).all()


@pytest.mark.parametrize("wide", [False, True])
def test_rows_that_do_not_see_a_key_are_untouched_by_it(ops, dev, wide):
    """A later token's K or V that is not finite reaches the rows that see it, and no earlier row."""
    import torch

    for D, what, val in ((64, "v", math.nan), (128, "v", math.inf), (64, "k", math.nan), (128, "k", math.inf)):
        q, kp, vp, table, out = _run_attention(ops, dev, [70, 50], 4, 8, 2, D, 16, wide=wide)
        lens = _ints([70, 50], dev)
        page, slot = int(table[0, 68 // 16]), 68 % 16
        q[0, :, :, 0] = 1.0  # a K of +inf then scores +inf, not NaN
        ref = ops.paged_attention(q, kp, vp, table, lens)
        (vp if what == "v" else kp)[page, slot, :, 0] = val
        got = ops.paged_attention(q, kp, vp, table, lens)
        assert torch.equal(got[0, :2], ref[0, :2]) and torch.equal(got[1], ref[1])
        bad = got[0, 2:]
        if what == "v":
            assert not torch.isfinite(bad[..., 0]).any() and torch.equal(bad[..., 1:], ref[0, 2:, :, 1:])
        else:
            assert torch.isnan(bad).all()


@pytest.mark.parametrize("key", [0, 7, 8, 100, 199])
@pytest.mark.parametrize("val", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("wide", [False, True])
def test_scores_without_a_softmax(ops, dev, key, val, wide):
    """A score of NaN or +inf makes its row NaN wherever it lies; one of -inf has no weight."""
    import torch

    q, kp, vp, table, out = _run_attention(ops, dev, [200, 200], 1, 4, 2, 128, 16, wide=wide)
    q[:, :, :, 3] = 1.0
    kp[int(table[1, key // 16]), key % 16, 1, 3] = val
    got = ops.paged_attention(q, kp, vp, table, _ints([200, 200], dev))
    if val == -math.inf:
        assert torch.isfinite(got).all()
    else:
        assert torch.isnan(got[1, 0, 2:]).all()
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1, 0, :2]).all()


@pytest.mark.parametrize("wide", [False, True])
def test_bad_pages_and_lengths(ops, dev, wide):
    """A page that is none of the cache, or a length past the table: that request's rows are NaN, no other's."""
    import torch

    q, kp, vp, table, out = _run_attention(ops, dev, [300, 280, 260, 40], 1, 8, 2, 64, 16, wide=wide)
    tab, lens = table.clone(), _ints([300, 280, 10 ** 9, -4], dev)
    tab[0, 7] = kp.shape[0]
    tab[3, 0] = 10 ** 9  # of a request without keys: never looked at
    got = ops.paged_attention(q, kp, vp, tab, lens)
    assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all() and (got[3] == 0).all()
    assert torch.equal(got[1], out[1]) or (got[1].float() - out[1].float()).abs().max() < 2e-2
    tab = table.clone()
    tab[1, 3] = -1
    assert torch.isnan(ops.paged_attention(q, kp, vp, tab, _ints([300, 280, 260, 40], dev))[1]).all()
    # a cache without pages, a table without room
    none = kp[:0]
    assert (ops.paged_attention(q, none, none, table, _ints([0] * 4, dev)) == 0).all()
    assert torch.isnan(ops.paged_attention(q, none, none, table, _ints([5] * 4, dev))).all()
    got = ops.paged_attention(q, kp, vp, table[:, :0], _ints([0, 1, 0, 0], dev))
    assert torch.isnan(got[1]).all() and (got[[0, 2, 3]] == 0).all()


def test_cache_past_32_bits(ops, dev):
    """Element offsets above 2^32 and byte offsets above 2^33, for both entries."""
    import torch

    size, D, step = 16, 64, 1 << 31  # elements between pages
    store = torch.empty(2 * step + 2 * size * D, dtype=torch.bfloat16, device=dev)
    kp = store.as_strided((3, size, 1, D), (step, D, D, 1))
    vp = store.as_strided((3, size, 1, D), (step, D, D, 1), size * D)
    r = rng(3)
    q, k, v = (_rand(r, (40, 1, D), "bf16", dev) for _ in range(3))
    table = _ints([[2, 0, 1]], dev)
    got = ops.paged_append(q, k, v, kp, vp, table, _ints([0], dev))
    assert torch.equal(got, q)
    out = ops.paged_attention(q[-1:], kp, vp, table, _ints([40], dev))
    torch.cuda.synchronize()
    _check_attention(out[:, None], q[-1:, None], kp, vp, table, [40], "bf16")


def test_results_repeat_and_survive_capture(ops, dev):
    """Equal bits each time; a captured step follows lengths, tables and tokens that change; two graphs at once."""
    import torch

    r = rng(9)
    lens = [900, 33, 2500]
    kp, vp, table, _ = _pages(r, [n + 8 for n in lens], 16, 2, 128, "bf16", dev)
    rope = ops.RotaryAxes(128, (64,), device=dev)
    w = _rand(r, (128,), "bf16", dev, 0.1, 1.0)
    q, k, v = (_rand(r, (3, h, 128), "bf16", dev) for h in (8, 2, 2))
    held = _ints(lens, dev)
    total = held + 1

    def step():
        got = ops.paged_append(q, k, v, kp, vp, table, held, rope=rope, q_weight=w, k_weight=w)
        return ops.paged_attention(got, kp, vp, table, total)
    first = step()
    assert all(torch.equal(step(), first) for _ in range(5))
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step())
        graphs.append(g)
    for n in ([900, 33, 2500], [5, 0, 17]):
        held.copy_(_ints(n, dev))
        total.copy_(held + 1)
        q.copy_(_rand(r, q.shape, "bf16", dev))
        want = step()
        torch.cuda.synchronize()
        for _ in range(3):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_another_stream(ops, dev):
    import torch

    q, kp, vp, table, out = _run_attention(ops, dev, [5000, 4000], 1, 16, 4, 128, 16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.paged_attention(q, kp, vp, table, _ints([5000, 4000], dev))
    s.synchronize()
    assert torch.equal(got, out)


def test_tokens_decoded_one_by_one(ops, dev):
    """Append and attention together, token by token and in stretches, against attention over the whole sequence."""
    import torch

    r = rng(21)
    B, L, Hq, Hkv, D, size = 3, 45, 4, 2, 64, 16
    rope = _rope(ops, D, (8, 12, 12), "half", 10000.0, dev)
    q, k, v = (_rand(r, (B, L, h, D), "bf16", dev) for h in (Hq, Hkv, Hkv))
    qw, kw = (_rand(r, (D,), "bf16", dev, 0.2, 1.0) for _ in range(2))
    pos = _ints(r.integers(0, 500, (B, L, 3)).tolist(), dev)
    kp, vp, table, _ = _pages(r, [L] * B, size, Hkv, D, "bf16", dev, fill=float("nan"))
    at = 0
    for n in (1, 20, 1, 1, 5, 16, 1):
        held = _ints([at] * B, dev)
        rows = slice(at, at + n)
        got = ops.paged_append(*(t[:, rows].reshape(B * n, -1, D) for t in (q, k, v)), kp, vp, table, held, rope=rope,
                               positions=pos[:, rows].reshape(B * n, 3), q_weight=qw, k_weight=kw)
        out = ops.paged_attention(got.view(B, n, Hq, D), kp, vp, table, held + n)
        at += n
        for b in range(B):
            kk = _turned(k[b, :at], kw, rope, pos[b, :at], 1e-6)[0].to(torch.bfloat16)
            assert torch.isfinite(out).all()
            # (a key or query may round the other way at a tie of the f32 norm: one step of it moves a score by
            # up to 2^-8 |q| |k| / sqrt(D) / sqrt(D) a pair, 2e-3 for a handful of elements)
            o, mag = _want(got.view(B, n, Hq, D)[b], kk, v[b, :at], at, D ** -0.5)
            bound = U["bf16"] * o.abs() + (4e-3 + 1.6e-4) * mag + 1e-7
            assert ((out[b].double() - o).abs() <= bound).all()
    assert at == L


def test_front_end_refuses(pkg, ops, dev):
    """The library's refusals come through the native calls with its words, each argument in its place."""
    import torch

    E = pkg._lib.L3dError

    def z(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=dev)
    q, kv, pages, table, held = z(2, 4, 64), z(2, 2, 64), z(3, 16, 2, 64), z(2, 1, dtype=torch.int32), z(2, dtype=torch.int32)
    ok = dict(q=q, k=kv, v=kv, k_pages=pages, v_pages=pages.clone(), table=table, held=held)
    assert ops.paged_append(**ok).shape == q.shape
    for over, word in ((dict(q=q.float()), "BF16"), (dict(k=kv[:1]), "k and v"), (dict(v=kv[:, :1]), "k and v"),
                       (dict(k_pages=pages[:2]), "k_pages and v_pages"), (dict(table=held), "table"),
                       (dict(held=held[:1]), "held"), (dict(offsets=held), "offsets"), (dict(q_weight=z(64)), "together"),
                       (dict(q_weight=z(64), k_weight=z(63)), "k_weight"), (dict(out=q[:1]), "q_out"), (dict(eps=-1.0), "eps")):
        with pytest.raises(E, match=word):
            ops.paged_append(**(ok | over))
    ok = dict(q=q, k_pages=pages, v_pages=pages, table=table, lengths=held)
    assert (ops.paged_attention(**ok) == 0).all()
    for over, word in ((dict(q=q[None, None]), r"\[B, N, H, D\]"), (dict(v_pages=pages[:2]), "k_pages and v_pages"),
                       (dict(table=table[:1]), "table"), (dict(lengths=held[:1]), "lengths"), (dict(out=q[:1]), "out"),
                       (dict(scale=0.0), "scale"), (dict(table=held), "table"), (dict(k_pages=kv, v_pages=kv), r"\[B, N, H, D\]")):
        with pytest.raises(E, match=word):
            ops.paged_attention(**(ok | over))
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    ok = dict(q=q, k=kv, v=kv, k_offsets=off)
    assert ops.cross_attention(**ok).shape == q.shape
    for over, word in ((dict(v=kv[:1]), "k and v"), (dict(k_offsets=off.float()), "k_offsets"), (dict(q_offsets=off[:2]), "q_offsets"),
                       (dict(k_offsets=off[None]), "k_offsets"), (dict(scale=-1.0), "scale"), (dict(out=q[:, :2]), "out"),
                       (dict(q=q[0]), "Tq, Hq, D"), (dict(k=kv[0], v=kv[0]), "Tk, Hkv, D")):
        with pytest.raises(E, match=word):
            ops.cross_attention(**(ok | over))
    for f, args in ((ops.paged_append, (q, kv.cpu(), kv, pages, pages, table, held)), (ops.paged_attention, (q, pages, pages, table.cpu(), held)),
                    (ops.cross_attention, (q, kv, kv, off.cpu()))):
        with pytest.raises(ValueError, match="CUDA"):
            f(*args)


@pytest.mark.parametrize("wide", [False, True])
def test_pages_shared_between_requests_and_caches_laid_out_unlike(ops, dev, wide):
    """Requests whose first pages are the same ones; keys by slot, values by head; tables with rows apart."""
    import torch

    r = rng(31)
    kp = _rand(r, (9, 16, 2, 64), "bf16", dev)
    vp = _rand(r, (9, 2, 16, 64), "bf16", dev).transpose(1, 2)
    tab = torch.full((3, 800 if wide else 20), 10 ** 6, dtype=torch.int32, device=dev)
    tab[:, 1:6] = _ints([[4, 0, 7, 2, 8], [4, 0, 7, 1, 3], [4, 5, 6, 6, 6]], dev)
    lens = [80, 61, 47]
    q = _rand(r, (3, 2, 4, 64), "bf16", dev)
    table = tab[:, 1:] if wide else tab[:, 1:6]
    out = ops.paged_attention(q, kp, vp, table, _ints(lens, dev), check=True)
    _check_attention(out, q, kp, vp, table, lens, "bf16")


def test_elements_past_32_bits_without_keys(ops, dev):
    """2^31 elements of a request without keys come out zero; of the other one the last row sees a key."""
    import torch

    N, H, D = 16384, 1024, 128
    q = torch.full((2, N, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    k, v = (_rand(rng(i), (1, 16, 1, D), "bf16", dev) for i in range(2))
    table = torch.zeros((2, 1), dtype=torch.int32, device=dev)
    ops.paged_attention(q, k, v, table, _ints([0, 1], dev), out=q, check=True)
    assert not q[0].any() and not q[1, :-1].any()
    assert torch.equal(q[1, -1], v[0, 0].expand(H, D))


def test_append_and_attend_in_place(ops, dev):
    """The queries may be written over: append's into the projection's rows, the attention's output over its queries."""
    import torch

    for lens in ([40, 7], [3000, 900]):
        q, kp, vp, table, out = _run_attention(ops, dev, lens, 1, 8, 2, 64, 16, wide=lens[0] > 100)
        got = q.clone()
        assert ops.paged_attention(got, kp, vp, table, _ints(lens, dev), out=got) is got
        assert torch.equal(got, out)
