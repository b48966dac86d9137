"""GPU parity: attention over a shared prefix and own keys
(l3d_shared_prefix_attention) against softmax in f64 on the same inputs.

Bound: the probabilities rounded to the input type (u = 2^-8 bf16, 2^-11 f16,
of sum p |v|; f16 below 2^-14 of the row's largest loses up to 2^-25 each), the
f32 scores and exponentials (4e-4 of sum p |v|: 1e-5 from the scores, 7.5e-5
twice from the polynomial exponential, the sums), and the output's rounding
(u |o|)."""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _rand(r, shape, dt, dev, std=1.0):
    import torch

    t = torch.from_numpy((std * r.standard_normal(shape)).astype(np.float32)).to(dev)
    return t.to(torch.bfloat16 if dt == "bf16" else torch.float16)


def _check(q, pk, pv, k, v, lens, causal, scale, out, dt):
    """out against the definition, per (batch, key head) in f64."""
    import torch

    B, Hq, N, D = q.shape
    H = pk.shape[0]
    G, P = Hq // H, pk.shape[1]
    assert out.shape == q.shape and out.dtype == q.dtype
    for b in range(B):
        n = 0 if k is None else int(min(max(lens[b], 0), k.shape[2]))
        for h in range(H):
            kk, vv = pk[h].double(), pv[h].double()
            if k is not None:
                kk, vv = torch.cat([kk, k[b, h, :n].double()]), torch.cat([vv, v[b, h, :n].double()])
            s = (q[b, h * G:(h + 1) * G].double() @ kk.T) * scale
            if causal:
                key = torch.arange(P + n, device=q.device) - P
                row = torch.arange(N, device=q.device)
                future = key[None] > (n - N + row)[:, None]  # of the own keys; the prefix is seen by every row
                s = s.masked_fill(future & (key >= 0)[None], float("-inf"))
            m = s.amax(-1, keepdim=True) if P + n else s.new_zeros(G, N, 1)
            p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
            l = p.sum(-1, keepdim=True)
            p = torch.where(l > 0, p / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(p))
            want = p @ vv
            mag = p @ vv.abs()
            bound = mag * (U[dt] + 4e-4) + want.abs() * U[dt] + 1e-6
            if dt == "f16" and P + n:
                bound = bound + (P + n) * 2.0 ** -25 * vv.abs().amax()
            err = (out[b, h * G:(h + 1) * G].double() - want).abs()
            assert (err <= bound).all(), \
                f"b {b} h {h}: max err {err.max().item():.3e}, worst ratio {(err / bound).max().item():.2f}"


def _run(ops, dev, B, Hq, H, N, D, P, S, lens=None, causal=False, dt="bf16", layout="token", std=1.0,
         scale=None):
    import torch

    r = rng(B * 1009 + N * 31 + P * 7 + S + D)
    if layout == "token":
        q = _rand(r, (B, N, Hq, D), dt, dev, std).transpose(1, 2)
        pk = _rand(r, (P, H, D), dt, dev, std).transpose(0, 1)
        pv = _rand(r, (P, H, D), dt, dev).transpose(0, 1)
    else:
        q, pk, pv = _rand(r, (B, Hq, N, D), dt, dev, std), _rand(r, (H, P, D), dt, dev, std), _rand(r, (H, P, D), dt, dev)
    k = v = lt = None
    if S:
        kv = _rand(r, (B, S, 2, H, D) if layout == "token" else (B, H, S, 2, D), dt, dev, std)
        k, v = (kv[:, :, i].transpose(1, 2) if layout == "token" else kv[:, :, :, i] for i in (0, 1))
        if lens is not None:
            lt = torch.tensor(lens, device=dev, dtype=torch.int32 if B % 2 else torch.int64)
            for b, n in enumerate(lens):  # what lies past an element's keys is not its concern
                kv[b, max(n, 0):] = float("nan") if layout == "token" else kv[b, max(n, 0):]
                if layout != "token":
                    kv[b, :, max(n, 0):] = float("inf")
    out = ops.shared_prefix_attention(q, pk, pv, k, v, lt, causal=causal, scale=scale)
    torch.cuda.synchronize()
    full = [S] * B if lens is None else lens
    _check(q, pk, pv, k, v, full, causal, D ** -0.5 if scale is None else scale, out, dt)
    return q, pk, pv, k, v, lt, out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,Hq,H,N,P,S,lens,causal", [
    (1, 1, 1, 1, 1, 0, None, False),
    (2, 4, 2, 1, 130, 40, [40, 7], False),              # one token per request
    (5, 8, 2, 1, 1029, 300, [300, 0, 1, 128, 129], False),
    (3, 6, 3, 5, 257, 77, [77, 5, 2], True),            # a few tokens; the last sees fewer than its rows
    (3, 3, 3, 200, 100, 0, None, False),                # cross attention alone
    (2, 4, 2, 300, 383, 300, [300, 211], False),        # joint attention, ragged
    (2, 2, 2, 270, 65, 270, [270, 100], True),          # causal over several tiles
    (1, 2, 1, 700, 500, 700, None, True),
    (7, 2, 2, 33, 129, 1, [1, 0, 1, 0, 1, 1, 0], False),
    (40, 16, 2, 1, 2000, 64, list(range(25, 65)), True),
])
def test_shared_prefix_attention(ops, dev, B, Hq, H, N, P, S, lens, causal, dt, D):
    _run(ops, dev, B, Hq, H, N, D, P, S, lens, causal, dt, layout="token" if (B + N) % 2 else "head")


@pytest.mark.parametrize("P", [1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 640, 5000])
def test_prefix_lengths(ops, dev, P):
    _run(ops, dev, 3, 4, 2, 2, 128, P, 130, [130, 64, 1], False)


@pytest.mark.parametrize("N", [1, 2, 16, 63, 64, 65, 127, 128, 129, 255, 256, 257, 513])
@pytest.mark.parametrize("causal", [False, True])
def test_row_counts(ops, dev, N, causal):
    _run(ops, dev, 2, 2, 1, N, 64, 190, 600, [600, 333], causal)


@pytest.mark.parametrize("B,Hq,H,N,D,P,S,causal", [
    (8, 16, 16, 300, 128, 1370, 300, False),   # prefix and own keys in one item
    (4, 12, 12, 128, 128, 1370, 500, True),
    (2, 16, 16, 200, 64, 1370, 900, False),    # in parts
    (8, 4, 4, 2049, 128, 1370, 0, False),      # several rounds of items
    (20, 4, 2, 40, 64, 9000, 70, True),        # prefix items apart from own ones
    (3, 4, 4, 1500, 128, 2, 590, True),
    (5, 8, 1, 33, 64, 0, 333, True),
])
def test_divisions_into_items(ops, dev, B, Hq, H, N, D, P, S, causal):
    lens = [S - (S * b) // B if not causal else max(min(N, S), S - 7 * b) for b in range(B)] if S else None
    _run(ops, dev, B, Hq, H, N, D, P, S, lens, causal)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("N", [1, 300])
def test_rows_without_keys_are_zero(ops, dev, N, dt):
    """No prefix and no own keys, and causal rows from before the element's first key."""
    import torch

    r = rng(N)
    q = _rand(r, (3, 2, N, 64), dt, dev)
    pk = torch.empty(2, 0, 64, device=dev, dtype=q.dtype)
    assert not ops.shared_prefix_attention(q, pk, pk).any()
    k = torch.full((3, 2, 9, 64), float("nan"), device=dev, dtype=q.dtype)
    k[1, :, :4] = _rand(r, (2, 4, 64), dt, dev)
    lens = torch.tensor([0, 4, -5], device=dev, dtype=torch.int32)
    out = ops.shared_prefix_attention(q, pk, pk, k, k, lens, causal=True)
    torch.cuda.synchronize()
    assert not out[0].any() and not out[2].any()
    _check(q, pk, pk, k, k, [0, 4, 0], True, 0.125, out, dt)
    if N > 4:
        assert not out[1, :, :N - 4].any()


@pytest.mark.parametrize("N", [1, 140])
def test_sharp_and_rising_scores(ops, dev, N):
    """Scores of large magnitude: the running maximum moves between tiles and between parts."""
    _run(ops, dev, 2, 4, 2, N, 128, 900, 300, [300, 45], std=3.0)
    _run(ops, dev, 2, 4, 2, N, 64, 900, 300, [300, 45], std=3.0, dt="f16")


@pytest.mark.parametrize("N", [1, 150])
def test_equals_attention_over_copies(ops, dev, N):
    """The prefix copied into every element and attended to as one sequence."""
    import torch

    q, pk, pv, k, v, _, out = _run(ops, dev, 3, 4, 4, N, 128, 200, 56)
    kk = torch.cat([pk.expand(3, -1, -1, -1), k], 2).contiguous()
    vv = torch.cat([pv.expand(3, -1, -1, -1), v], 2).contiguous()
    want = ops.attention(q, kk, vv)
    assert ((out - want).float().norm() / want.float().norm()).item() < 5e-3


def test_lengths_are_clamped(ops, dev):
    import torch

    q, pk, pv, k, v, _, out = _run(ops, dev, 2, 2, 1, 3, 64, 50, 20, [20, 0])
    lens = torch.tensor([2 ** 40, -(2 ** 40)], device=dev)
    k2, v2 = k.clone(), v.clone()
    assert torch.equal(ops.shared_prefix_attention(q, pk, pv, k2, v2, lens), out)


def test_strided_output(ops, dev):
    import torch

    q, pk, pv, k, v, lt, want = _run(ops, dev, 2, 4, 2, 9, 64, 300, 30, [30, 11])
    buf = torch.full((2, 9, 4, 128), 7.0, device=dev, dtype=torch.bfloat16)
    ops.shared_prefix_attention(q, pk, pv, k, v, lt, out=buf[..., 64:].transpose(1, 2))
    assert torch.equal(buf[..., 64:].transpose(1, 2), want)
    assert (buf[..., :64] == 7).all()


@pytest.mark.parametrize("N", [1, 200])
def test_offsets_past_32_bits(ops, dev, N):
    """Own keys and prefix rows that lie more than 2^31 elements into their storage."""
    import torch

    r = rng(11)
    big = torch.empty((1 << 31) + (1 << 24), device=dev, dtype=torch.bfloat16)
    D, P, S, step = 64, 33, 20, 1 << 25
    pk = big.as_strided((2, P, D), (D, step, 1), 0)           # rows 2^25 apart: the last passes 2^30
    pv = big.as_strided((2, P, D), (D, step, 1), 2 * D)
    k = big.as_strided((2, 2, S, D), ((1 << 31) - 4096, 1 << 16, 256, 1), 1 << 20)
    v = big.as_strided((2, 2, S, D), ((1 << 31) - 4096, 1 << 16, 256, 1), (1 << 20) + 128)
    for t in (pk, pv, k, v):
        t.copy_(_rand(r, t.shape, "bf16", dev))
    q = _rand(r, (2, 4, N, D), "bf16", dev)
    out = ops.shared_prefix_attention(q, pk, pv, k, v)
    torch.cuda.synchronize()
    _check(q, pk, pv, k, v, [S, S], False, 0.125, out, "bf16")


@pytest.mark.parametrize("N", [1, 300])
def test_other_stream_and_graph(ops, dev, N):
    import torch

    q, pk, pv, k, v, lt, want = _run(ops, dev, 4, 8, 2, N, 128, 1000, 90, [90, 1, 0, 60], True)
    for _ in range(3):  # the same bits on every call
        assert torch.equal(ops.shared_prefix_attention(q, pk, pv, k, v, lt, causal=True), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.shared_prefix_attention(q, pk, pv, k, v, lt, causal=True)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            kept = ops.shared_prefix_attention(q, pk, pv, k, v, lt, causal=True)
        g.replay()
        g.replay()
    s.synchronize()
    assert torch.equal(other, want) and torch.equal(kept, want)


def test_refusals(pkg, ops, dev):
    import torch

    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, device=dev, dtype=dt)  # noqa: E731
    ok = dict(q=z(2, 4, 3, 64), prefix_k=z(2, 9, 64), prefix_v=z(2, 9, 64), k=z(2, 2, 5, 64), v=z(2, 2, 5, 64))
    bad = [
        (dict(q=z(2, 3, 3, 64)), "multiple"), (dict(q=z(2, 4, 3, 96)), "64 or 128"),
        (dict(prefix_v=z(2, 8, 64)), "prefix"), (dict(v=z(2, 2, 6, 64)), r"\[B, Hkv, S, D\]"),
        (dict(v=None), "together"), (dict(k=None, v=None, causal=True), "own keys"),
        (dict(lengths=torch.zeros(3, device=dev, dtype=torch.int32)), "contiguous"),
        (dict(lengths=torch.zeros(2, device=dev)), "I32 or I64"),
        (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
        (dict(k=z(2, 2, 5, 64, dt=torch.float16)), "BF16"), (dict(q=z(2, 4, 3, 64, dt=torch.float32)), "BF16"),
        (dict(prefix_k=z(2, 9, 68)[..., 4:]), "aligned|multiples"),
        (dict(out=z(2, 4, 4, 64)), "out"),
        (dict(prefix_k=z(2, 64, 9).transpose(1, 2)), "contiguous"),
    ]
    for kw, match in bad:
        with pytest.raises(pkg._lib.L3dError, match=match):
            ops.shared_prefix_attention(**(ok | kw))
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_prefix_attention(**(ok | dict(q=ok["q"].cpu())))
    assert ops.shared_prefix_attention(z(0, 4, 3, 64), ok["prefix_k"], ok["prefix_v"]).shape == (0, 4, 3, 64)
    assert ops.shared_prefix_attention(z(2, 4, 0, 64), ok["prefix_k"], ok["prefix_v"]).shape == (2, 4, 0, 64)


@pytest.mark.parametrize("N", [1, 150])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("value", ["nan", "inf"])
def test_bad_key_is_seen_wherever_it_lies(ops, dev, value, own, D, dt, N):
    """A key whose score is NaN or +inf makes the rows that see it NaN, at each of 16
    consecutive places of a tile, and no other row differs."""
    import torch

    r = rng(N + D)
    q, pk, pv, k, v = (_rand(r, s, dt, dev) for s in ((2, 4, N, D), (2, 100, D), (2, 100, D), (2, 2, 70, D), (2, 2, 70, D)))
    q[..., 0] = 1
    want = ops.shared_prefix_attention(q, pk, pv, k, v)
    missed = []
    for at in range(16, 32):
        k2, pk2 = k.clone(), pk.clone()
        (k2[1] if own else pk2)[1, at, 0] = float(value)
        got = ops.shared_prefix_attention(q, pk2, pv, k2, v)
        touched = torch.zeros_like(got, dtype=torch.bool)
        touched[1 if own else slice(None), 2:] = True
        assert torch.equal(got[~touched], want[~touched])
        if not torch.isnan(got[touched]).all():
            missed.append(at)
    assert not missed


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [40, 200])
def test_masked_values_of_any_size_add_nothing(ops, dev, N, D):
    """V of a key that a causal row does not see, at the end of bf16's range, at each
    place of a tile: the rows before it keep their bits."""
    import torch

    r = rng(N + D)
    q, pk, pv, k, v = (_rand(r, s, "bf16", dev) for s in ((1, 2, N, D), (2, 30, D), (2, 30, D), (1, 2, N, D), (1, 2, N, D)))
    want = ops.shared_prefix_attention(q, pk, pv, k, v, causal=True)
    changed = []
    for at in range(1, 40):
        v2 = v.clone()
        v2[:, :, at] = 3e38
        got = ops.shared_prefix_attention(q, pk, pv, k, v2, causal=True)
        if not torch.equal(got[:, :, :at], want[:, :, :at]):
            changed.append(at)
    assert not changed
