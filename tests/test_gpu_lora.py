"""GPU parity: a projection with low-rank adapters of many requests
(l3d_lora_linear) against the f64 sum of the same bf16 operands.

Bounds: f32 accumulation of both products (2e-5 of the sum of the terms'
magnitudes, as for the dense linear); A x rounded to bf16 before the second
product (2^-9 of its terms; 2^-17 where y is F32 and it enters as two bf16
parts), times the activation's largest derivative (< 1.13); for a bf16 y its
rounding (2^-8) and the 16-bit activation forms (3e-4 |z|)."""
import numpy as np
import pytest

from conftest import rng
from test_gpu_qlinear import _act_ref

pytestmark = pytest.mark.gpu


def _case(ops, dev, M, N, K, ranks, ids, act=None, res=False, gate=False, ydt="bf16", bias=True,
          seed=0, x=None):
    import torch

    r = rng(700 + seed + M + N + K)

    def up(a, dt=torch.bfloat16):
        t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(dev).to(dt)
        return t, t.float().cpu().numpy().astype(np.float64)

    xt, xv = up(r.standard_normal((M, K)))
    if x is not None:
        x.copy_(xt)
        xt = x
    wt, wv = up(r.standard_normal((N, K)) / np.sqrt(K))
    ab = [(up(r.standard_normal((k, K)) / np.sqrt(K)), up(0.5 * r.standard_normal((N, k)) / np.sqrt(k)))
          for k in ranks]
    scales = [0.5 + 0.5 * i for i in range(len(ranks))]
    ad = ops.LoraAdapters([a[0] for a, _ in ab], [b[0] for _, b in ab], scales)
    z, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    bt = None
    if bias:
        bt, bv = up(0.1 * r.standard_normal(N), torch.float32)
        z = z + bv
    ids = np.asarray(ids)
    per = np.repeat(ids, M // ids.size)
    low = np.zeros_like(z)
    for i, ((_, av), (_, bv)) in enumerate(ab):
        rows = per == i
        z[rows] += scales[i] * (xv[rows] @ av.T) @ bv.T
        mag[rows] += scales[i] * (np.abs(xv[rows]) @ np.abs(av).T) @ np.abs(bv).T
        low[rows] += scales[i] * np.abs(xv[rows] @ av.T) @ np.abs(bv).T
    bound = 1.13 * (2e-5 * mag + low * (2.0 ** -9 if ydt == "bf16" else 2.0 ** -17)) + 1e-6
    ref = _act_ref(act, z)
    tdt = torch.float32 if ydt == "f32" else torch.bfloat16
    kw = {"act": act, "bias": bt, "out_dtype": tdt}
    if res:
        rt, rv = up(r.standard_normal((M, N)), tdt)
        gv = 1.0
        if gate:
            kw["gate"], gv = up(0.5 + r.random(N), torch.float32)
        ref = rv + gv * ref
        bound = bound * np.max(np.abs(gv))
        kw.update(residual=rt, out=rt)
    if ydt == "bf16":
        bound = bound + np.abs(ref) * 2.0 ** -8 + (3e-4 * np.abs(z) if act else 0.0)
    else:
        bound = bound + 1e-6 * np.abs(ref)
    got = ops.lora_linear(xt, wt, ad, torch.from_numpy(ids).to(dev), **kw)
    torch.cuda.synchronize()
    err = np.abs(got.float().cpu().numpy() - ref)
    assert np.all(err <= bound), f"max err {err.max():.3e}, worst ratio {(err / bound).max():.2f}"
    return ad, xt, wt, got


@pytest.mark.parametrize("M,N,K,ranks,A_ids", [
    (1, 64, 64, [16], "all0"),
    (1, 2048, 1024, [8, 16], "row"),
    (3, 77, 72, [1, 5], "row"),
    (16, 2048, 2048, [16] * 8, "row"),
    (16, 1000, 264, [4, 64, 16], "row"),
    (64, 512, 520, [64, 32, 16] * 11, "row"),     # more adapters than fit one stage
    (127, 200, 128, [24] * 40, "row"),
    (129, 384, 256, [48, 3], "row"),
    (300, 264, 520, [33, 128], "request"),
    (640, 1024, 1024, [256, 16], "row"),          # the largest rank
    (1000, 520, 328, [16, 8, 64], "scene"),
    (1, 8, 8, [1], "none"),
])
@pytest.mark.parametrize("ydt", ["bf16", "f32"])
def test_lora_linear(ops, dev, M, N, K, ranks, A_ids, ydt):
    r, A = rng(M * 13 + N), len(ranks)
    if A_ids == "all0":
        ids = np.zeros(M, np.int64)
    elif A_ids == "none":
        ids = np.full(M, -1, np.int64)
    elif A_ids == "request":  # M / 3 rows per id
        ids = np.asarray([1, -1, 0], np.int32)
    elif A_ids == "scene":
        ids = np.sort(r.integers(-1, A, M)).astype(np.int32)
    else:  # any adapter, or none (on either side of the range), for each row
        ids = r.integers(-2, A + 1, M).astype(np.int64)
    _case(ops, dev, M, N, K, ranks, ids, ydt=ydt)


@pytest.mark.parametrize("M,N,K", [(5, 136, 512), (200, 300, 256), (1500, 768, 512)])
@pytest.mark.parametrize("act,res,gate,ydt,bias", [
    ("gelu_erf", False, False, "bf16", True),
    ("gelu", True, True, "bf16", True),
    ("silu", True, False, "f32", False),
    (None, True, True, "f32", True),
    (None, True, True, "bf16", False),
])
def test_lora_linear_epilogue(ops, dev, M, N, K, act, res, gate, ydt, bias):
    ids = rng(M).integers(-1, 3, M).astype(np.int32)
    _case(ops, dev, M, N, K, [16, 32, 8], ids, act, res, gate, ydt, bias)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 128, 255, 257, 512, 1025])
def test_lora_linear_row_counts(ops, dev, M):
    _case(ops, dev, M, 320, 320, [16, 32], rng(M).integers(-1, 2, M).astype(np.int32), "silu")


def test_lora_linear_many_tiles(ops, dev):
    """More tiles than blocks: each block works through several, with other adapters in each."""
    _case(ops, dev, 5000, 2560, 192, [16, 32, 64, 16], rng(9).integers(-1, 4, 5000).astype(np.int32))


@pytest.mark.parametrize("M,N,K,ranks,kind", [
    (2369, 96, 264, [16, 48], "scene"),     # around the row count where A x changes its kernel
    (2368, 96, 264, [16, 48], "scene"),
    (2500, 77, 136, [256, 8], "scene"),
    (2600, 40, 72, [16] * 20, "row"),       # many adapters in every tile
    (12001, 64, 520, [64], "request"),
])
def test_lora_linear_many_rows(ops, dev, M, N, K, ranks, kind):
    A = len(ranks)
    ids = {"scene": lambda: np.sort(rng(M).integers(-1, A, M)), "row": lambda: rng(M).integers(-1, A, M),
           "request": lambda: np.asarray([0, -1, 0, -1, 0, 0, 0][:next(n for n in (7, 1) if M % n == 0)])}[kind]()
    _case(ops, dev, M, N, K, ranks, ids.astype(np.int32))


def test_lora_linear_strided_rows(ops, dev):
    """x and out as column ranges of wider matrices; nothing else is written."""
    import torch

    xw = torch.zeros(70, 512, device=dev, dtype=torch.bfloat16)
    ids = rng(3).integers(-1, 2, 70).astype(np.int32)
    ad, x, w, _ = _case(ops, dev, 70, 96, 256, [16, 16], ids, bias=False, x=xw[:, 128:384])
    wide = torch.full((70, 100), 7.0, device=dev, dtype=torch.bfloat16)  # rows of 200 bytes
    ops.lora_linear(x, w, ad, torch.from_numpy(ids).to(dev), out=wide[:, 2:98])
    want = ops.lora_linear(x, w, ad, torch.from_numpy(ids).to(dev))
    assert torch.equal(wide[:, 2:98], want)
    assert (wide[:, :2] == 7).all() and (wide[:, 98:] == 7).all()


def test_lora_linear_rows_are_independent(ops, dev):
    """A row's result depends on its own input and adapter alone: not on what
    other rows hold (even NaN), and equal on every call."""
    import torch

    ids = rng(4).integers(-1, 5, 200).astype(np.int32)
    ad, x, w, y = _case(ops, dev, 200, 512, 512, [16] * 5, ids, bias=False)
    t = torch.from_numpy(ids).to(dev)
    x2 = x.clone()
    x2[::2] = float("nan")
    got = ops.lora_linear(x2, w, ad, t)
    assert torch.equal(got[1::2], y[1::2]) and torch.isnan(got[::2]).all()
    for _ in range(3):
        assert torch.equal(ops.lora_linear(x, w, ad, t), y)


def test_lora_linear_without_adapters_is_linear(ops, dev):
    import torch

    ids = np.full(300, -1, np.int32)
    ad, x, w, y = _case(ops, dev, 300, 512, 512, [16], ids, bias=False)
    want = x.double() @ w.double().T
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-3).all()


def test_lora_linear_empty_and_shapes(ops, dev):
    import torch

    ad, x, w, _ = _case(ops, dev, 12, 64, 64, [16], np.zeros(12, np.int32), bias=False)
    none = torch.zeros(0, device=dev, dtype=torch.int32)
    assert ops.lora_linear(x[:0], w, ad, none).shape == (0, 64)
    y = ops.lora_linear(x.view(3, 4, 64), w, ad, torch.tensor([0, -1, 0], device=dev))
    assert y.shape == (3, 4, 64)
    assert torch.equal(y[0], ops.lora_linear(x[:4], w, ad, torch.zeros(4, device=dev, dtype=torch.int64)))


def test_lora_linear_other_stream_and_graph(ops, dev):
    import torch

    ids = rng(6).integers(-1, 2, 160).astype(np.int32)
    ad, x, w, y = _case(ops, dev, 160, 512, 512, [16, 32], ids, bias=False)
    t = torch.from_numpy(ids).to(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.lora_linear(x, w, ad, t)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            kept = ops.lora_linear(x, w, ad, t)
        g.replay()
        g.replay()
    s.synchronize()
    assert torch.equal(other, y) and torch.equal(kept, y)


def test_lora_linear_refusals(pkg, ops, dev):
    import torch

    ad, x, w, y = _case(ops, dev, 12, 64, 64, [16], np.zeros(12, np.int32), bias=False)
    t = torch.zeros(12, device=dev, dtype=torch.int32)
    bad = [
        (dict(x=x.float()), "BF16"), (dict(weight=w.float()), "BF16"),
        (dict(ids=t.float()), "I32 or I64"), (dict(ids=t[:5]), "divide evenly"),
        (dict(gate=torch.ones(64, device=dev)), "needs a residual"),
        (dict(bias=torch.ones(63, device=dev)), "bias"),
        (dict(residual=y.float()), "dtype"),
        (dict(weight=torch.zeros(32, 64, device=dev, dtype=torch.bfloat16)), "lora_b"),
        (dict(x=torch.zeros(12, 72, device=dev, dtype=torch.bfloat16)[:, 4:68]), "aligned"),
        (dict(out_dtype=torch.float16), "y must be"),
    ]
    for kw, match in bad:
        args = {"x": x, "weight": w, "adapters": ad, "ids": t} | kw
        with pytest.raises(pkg._lib.L3dError, match=match):
            ops.lora_linear(**args)
    with pytest.raises(ValueError, match="finite"):
        ops.LoraAdapters([torch.full((4, 64), float("inf"), device=dev)], [torch.zeros(64, 4, device=dev)])
    with pytest.raises(ValueError, match="expected"):
        ops.LoraAdapters([torch.zeros(4, 64, device=dev)], [torch.zeros(64, 5, device=dev)])
    with pytest.raises(ValueError):
        ops.LoraAdapters([], [])
    with pytest.raises(ValueError, match="CUDA"):
        ops.lora_linear(x.cpu(), w, ad, t)


@pytest.mark.parametrize("ydt", ["bf16", "f32"])
def test_lora_linear_stretches_of_rows(ops, dev, ydt):
    """Rows in stretches of 128 to 400, one adapter each: every block works through
    several row tiles with fewer slot stages than warps that fill them, and with
    other adapters from tile to tile.  Equal bits on every call."""
    import torch

    r, M = rng(21), 20000
    ids = np.concatenate([np.full(n, r.integers(-1, 40)) for n in r.integers(128, 401, 160)])[:M].astype(np.int32)
    assert ids.size == M
    ad, x, w, y = _case(ops, dev, M, 640, 128, [16] * 40, ids, bias=False, ydt=ydt)
    t = torch.from_numpy(ids).to(dev)
    for _ in range(20):
        assert torch.equal(ops.lora_linear(x, w, ad, t, out_dtype=y.dtype), y)


@pytest.mark.parametrize("M", [1, 40, 2368, 6000])
def test_lora_linear_without_adapters_leaves_nothing_running(pkg, ops, dev, M):
    """No row has an adapter, and the next operation on the stream gives every id a
    value and the workspace another use: the call is then done with both."""
    import torch

    ad, x, w, y = _case(ops, dev, M, 64, 1024, [64, 64], np.full(M, -1, np.int32), bias=False)
    t = torch.full((M,), -1, dtype=torch.int32, device=dev)
    need = pkg._lib.lib().l3d_lora_linear_workspace_size(M, ad.rank)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    out = torch.empty_like(y)
    for _ in range(20):
        t.fill_(-1)
        dx, dw, dt, do = pkg._lib.packs(x, w, t, out)
        pkg._lib.call("l3d_lora_linear", dx, dw, None, *ad._desc, dt, 0, None, None, do, ws.data_ptr(), need,
                      pkg._lib.stream_of(x))
        t.fill_(1)
        ws.fill_(7)
        torch.cuda.synchronize()
        assert (ws == 7).all() and torch.equal(out, y)


def _one_row_apart(dev, M, rank, row):
    """x zero but for one row; operands [M, 64], [48, 64], [rank, 64], [48, rank], all zero."""
    import torch

    z = lambda *s: torch.zeros(s, device=dev, dtype=torch.bfloat16)  # noqa: E731
    return z(M, 64), z(48, 64), z(rank, 64), z(48, rank), torch.zeros(M, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("M", [5, 2400])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_lora_linear_infinite_row(ops, dev, M, sign):
    """An infinite element of x under positive weights: the row is infinite, not NaN."""
    import torch

    x, w, a, b, ids = _one_row_apart(dev, M, 16, 3)
    x.fill_(0.5)
    w.fill_(0.25), a.fill_(0.125), b.fill_(0.5)
    x[3, 7] = sign * float("inf")
    y = ops.lora_linear(x, w, ops.LoraAdapters([a], [b]), ids)
    assert (y[3] == sign * float("inf")).all()
    assert torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()


@pytest.mark.parametrize("M", [5, 2400])
def test_lora_linear_a_x_at_the_end_of_the_range(ops, dev, M):
    """A x between bf16's largest value and f32's: two parts hold it to 2^-16."""
    import torch

    x, w, a, b, ids = _one_row_apart(dev, M, 16, 2)
    x[2, 0], x[2, 1] = 2.0 ** 127, 2.0 ** 119
    a[0, 0], a[0, 1] = 255 / 128, 1.25
    b[:, 0] = 2.0 ** -120
    y = ops.lora_linear(x, w, ops.LoraAdapters([a], [b]), ids, out_dtype=torch.float32)
    want = 255.0 + 1.25 * 2.0 ** -1  # 2^127 255/128 + 2^119 1.25, over 2^120
    assert ((y[2].double() - want).abs() <= want * 2.0 ** -16).all()
    assert not y[:2].any() and not y[3:].any()


@pytest.mark.parametrize("M", [5, 2400])
@pytest.mark.parametrize("rank", [1, 5, 33])
def test_lora_linear_infinite_row_and_padded_ranks(ops, dev, M, rank):
    """The ranks that an adapter is padded with take no part in an infinite row."""
    import torch

    x, w, a, b, ids = _one_row_apart(dev, M, rank, 3)
    x.fill_(0.5)
    w.fill_(0.25), a.fill_(0.125), b.fill_(0.5)
    x[3, 7] = float("inf")
    y = ops.lora_linear(x, w, ops.LoraAdapters([a, a.repeat(2, 1)], [b, b.repeat(1, 2)]), ids)
    assert (y[3] == float("inf")).all()
    assert torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("ydt", ["bf16", "f32"])
def test_lora_linear_tanh_gelu_in_its_tail(ops, dev, M, ydt):
    """The tanh GELU of z from -6 to 6, which the bias gives exactly: accurate relative
    to its value.  A bf16 y is the rounding of a value within 2e-5 of the exact one
    (an argument of the exponential up to 25 with a few f32 roundings), so it lies
    between the roundings of that range's ends; an f32 y has the formula 0.5 z (1 +
    tanh u) in f32, 2^-23 of |z| from its sum and 2e-6 of the value."""
    import torch

    N = 1024
    z = torch.linspace(-6, 6, N, device=dev)
    ad = ops.LoraAdapters([torch.zeros(1, 64, device=dev)], [torch.zeros(N, 1, device=dev)])
    x, w = (torch.zeros(n, 64, device=dev, dtype=torch.bfloat16) for n in (M, N))
    got = ops.lora_linear(x, w, ad, torch.zeros(M, dtype=torch.int32, device=dev), bias=z, act="gelu",
                          out_dtype=torch.float32 if ydt == "f32" else torch.bfloat16).double()
    zd = z.double()
    want = zd / (1 + torch.exp(-2 * (2 / np.pi) ** 0.5 * (zd + 0.044715 * zd ** 3)))
    if ydt == "bf16":
        lo, hi = (t.to(torch.bfloat16).double() for t in (want - 2e-5 * want.abs(), want + 2e-5 * want.abs()))
        assert ((got >= lo) & (got <= hi)).all()
    else:
        assert ((got - want).abs() <= zd.abs() * 2.0 ** -23 + want.abs() * 2e-6).all()


def test_lora_linear_refuses_rows_of_another_length(pkg, ops, dev):
    """A batch of rows that as many elements would fit otherwise is not cut anew."""
    import torch

    ad, x, w, _ = _case(ops, dev, 12, 64, 64, [16], np.zeros(12, np.int32), bias=False)
    one = torch.zeros(2, device=dev, dtype=torch.int32)
    z = lambda *s: torch.zeros(s, device=dev, dtype=torch.bfloat16)  # noqa: E731
    for kw, match in [(dict(x=z(2, 3, 128)), "x last dim"), (dict(x=z(2, 3, 32)), "x last dim"),
                      (dict(residual=z(2, 3, 128)), "residual"), (dict(out=z(2, 3, 32)), "y last dim"),
                      (dict(residual=z(2, 6, 32)), "leading dims")]:
        with pytest.raises((pkg._lib.L3dError, ValueError), match=match):
            ops.lora_linear(**({"x": z(2, 3, 64), "weight": w, "adapters": ad, "ids": one} | kw))
    r = torch.randn(2, 3, 64, device=dev).to(torch.bfloat16)
    x3 = x[:6].view(2, 3, 64)
    want = ops.lora_linear(x3, w, ad, one, residual=r)
    assert torch.equal(ops.lora_linear(x3, w, ad, one, residual=r.view(6, 64)), want)
    assert torch.equal(ops.lora_linear(x[:6], w, ad, one, residual=r), want.view(6, 64))


@pytest.mark.parametrize("M,N", [(1, 64), (33, 96), (129, 256), (300, 100), (2400, 512)])
@pytest.mark.parametrize("ydt", ["bf16", "f32"])
def test_lora_linear_residual_of_other_strides(ops, dev, M, N, ydt):
    """A residual in memory of its own, with rows of another stride than y's and a
    last row tile that is partly filled: the same bits as in place."""
    import torch

    ids = rng(M).integers(-1, 2, M).astype(np.int32)
    ad, x, w, _ = _case(ops, dev, M, N, 128, [16, 40], ids, bias=False, ydt=ydt)
    t, dt = torch.from_numpy(ids).to(dev), torch.float32 if ydt == "f32" else torch.bfloat16
    g = torch.Generator().manual_seed(M)
    res = torch.randn(M, N, generator=g).to(dev, dt)
    gate = torch.randn(N, generator=g).to(dev)
    y = res.clone()
    ops.lora_linear(x, w, ad, t, residual=y, gate=gate, out=y)
    wide = torch.zeros(M, N + 40, device=dev, dtype=dt)
    for off in (0, 8, 3):  # 3: not 16-byte aligned
        wide[:, off:off + N] = res
        got = ops.lora_linear(x, w, ad, t, residual=wide[:, off:off + N], gate=gate, out_dtype=dt)
        if off != 3 and N % 32 == 0:
            assert torch.equal(got, y)
        else:  # an unaligned row adds residual and gated product in one rounding, not two
            far = (got.double() - y.double()).abs() - 2.0 ** -22 * (y.double().abs() + res.double().abs())
            assert (far <= (2.0 ** -7 * y.double().abs() if ydt == "bf16" else 0.0)).all()
        assert torch.equal(wide[:, off:off + N], res)


@pytest.mark.parametrize("M", [1, 5, 130, 2369, 5000])
def test_lora_linear_holds_a_x_in_two_parts(ops, dev, M):
    """A x that needs 16 bits, picked out by B: y is exactly A x in f32, and its
    rounding in bf16, for either kernel that forms A x."""
    import torch

    K, N, ranks = 136, 256, (1, 40, 256)
    g = torch.Generator().manual_seed(M)
    z = lambda *s: torch.zeros(s, device=dev, dtype=torch.bfloat16)  # noqa: E731
    x, a, b, t = z(M, K), [], [], []
    x[:, 3], x[:, 135] = 1, 2.0 ** -9
    for r in ranks:
        hi, lo = 128 + torch.randint(0, 128, (r,), generator=g), torch.randint(0, 128, (r,), generator=g)
        a.append(z(r, K)), b.append(z(N, r))
        a[-1][:, 3], a[-1][:, 135] = hi.to(dev), lo.to(dev)
        pick = torch.arange(N) % r
        b[-1][torch.arange(N), pick] = 1
        t.append((hi + lo * 2.0 ** -9)[pick].to(dev, torch.float32))
    ids = torch.randint(-1, 3, (M,), generator=g).to(dev, torch.int32)
    want = torch.cat([torch.stack(t), torch.zeros(1, N, device=dev)])[ids.long()]
    ad = ops.LoraAdapters(a, b)
    assert torch.equal(ops.lora_linear(x, z(N, K), ad, ids, out_dtype=torch.float32), want)
    assert torch.equal(ops.lora_linear(x, z(N, K), ad, ids), want.to(torch.bfloat16))


@pytest.mark.parametrize("M,N,K,ranks,kind", [
    (2369, 96, 264, [16, 48], "scene"), (2500, 77, 136, [256, 8], "scene"), (2600, 40, 72, [16] * 20, "row"),
    (12001, 64, 520, [64], "scene"), (5000, 2560, 192, [16, 32, 64, 16], "row"),
])
def test_lora_linear_many_rows_in_f32(ops, dev, M, N, K, ranks, kind):
    """As the tests of many rows and tiles, with an output that does not round their errors away."""
    ids = rng(M).integers(-1, len(ranks), M).astype(np.int32)
    _case(ops, dev, M, N, K, ranks, np.sort(ids) if kind == "scene" else ids, ydt="f32")
