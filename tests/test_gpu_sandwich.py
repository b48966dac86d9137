"""GPU parity: the block seam with a norm on either side of the residual
(l3d_sandwich_residual_norm) against its definition in f64 on the same inputs
(the suite's tolerances: f32 1e-5, 16-bit max(2e-2, 2^-8 |ref|))."""
import numpy as np
import pytest

from conftest import assert_close, rng, to_dev

pytestmark = pytest.mark.gpu


def _norm(kind, v, w, b, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdims=True)
    v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
    v = v if w is None else v * w
    return v if b is None else v + b


def _ref(kind, x, h, pw, pb, g, a, w, b, sh, sc, post_eps, eps):
    def per(t):  # [C], [B, C] or [B, 1, C] against [B, T, C]
        return t if t.ndim == 1 else t.reshape(t.shape[0], 1, t.shape[-1])

    n = _norm(kind, h, pw, pb, post_eps)
    r = a * x + (n if g is None else per(g) * n)
    y = _norm(kind, r, w, b, eps)
    if sc is not None:
        y = y * (1 + per(sc))
    if sh is not None:
        y = y + per(sh)
    return r, y


def _run(ops, dev, B, T, C, kind, dt, vecs, seed=0, a=0.75, vdt=None, mean=0.3, **kw):
    import torch

    r = rng(900 + seed + B * T + C)
    x, xv = to_dev(r.standard_normal((B, T, C)), dt, dev)
    h, hv = to_dev(3 * r.standard_normal((B, T, C)) + mean, dt, dev)
    t, f = {}, {}
    shape = {"pw": (C,), "pb": (C,), "w": (C,), "b": (C,), "g": (C,), "sh": (C,), "sc": (C,)}
    for name, per in vecs.items():
        s = (B, C) if per == "BC" else (B, 1, C) if per == "B1C" else shape[name]
        one = 1.0 if name in ("pw", "w", "g") else 0.0
        t[name], f[name] = to_dev(one + 0.2 * r.standard_normal(s), vdt or dt, dev)
        f[name] = f[name].astype(np.float64)
    get = lambda d, k: d.get(k)  # noqa: E731
    ro, yo = ops.sandwich_residual_norm(x, h, post_weight=get(t, "pw"), post_bias=get(t, "pb"), gate=get(t, "g"),
                                        res_scale=a, weight=get(t, "w"), bias=get(t, "b"), shift=get(t, "sh"),
                                        scale=get(t, "sc"), norm=kind, eps=1e-5, post_eps=1e-6, **kw)
    torch.cuda.synchronize()
    rr, yr = _ref(kind, xv.astype(np.float64), hv.astype(np.float64), get(f, "pw"), get(f, "pb"), get(f, "g"), a,
                  get(f, "w"), get(f, "b"), get(f, "sh"), get(f, "sc"), 1e-6, 1e-5)
    assert_close(ro.float().cpu().numpy(), rr, dt, "r")
    if yo is not None:
        assert_close(yo.float().cpu().numpy(), yr, dt, "y")
    return x, h, ro, yo


ADA = {"pw": "C", "w": "C", "g": "BC", "sh": "B1C", "sc": "BC"}
AFFINE = {"pw": "C", "pb": "C", "w": "C", "b": "C", "g": "C"}


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("B,T,C", [
    (1, 1, 8), (2, 3, 1), (1, 5, 77), (3, 7, 64), (2, 9, 96), (2, 40, 1000), (1, 33, 1024), (3, 50, 1536),
    (2, 17, 2048), (1, 5, 4096), (2, 3, 8192), (1, 2, 16384), (1, 2, 20001), (1, 1, 24576),
])
def test_sandwich(ops, dev, B, T, C, kind, dt):
    _run(ops, dev, B, T, C, kind, dt, ADA if kind == "rms" else AFFINE)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("vecs", [{}, {"pw": "C"}, {"g": "BC"}, {"w": "C", "sc": "C"}, {"b": "C", "sh": "BC"},
                                  AFFINE | ADA])
@pytest.mark.parametrize("C", [256, 2048, 331])
def test_sandwich_optional_vectors(ops, dev, kind, vecs, C):
    _run(ops, dev, 3, 21, C, kind, "bf16", vecs, vdt="f32" if len(vecs) % 2 else None)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,C", [(4, 4000, 256), (2, 9000, 1024), (40, 77, 512), (1, 3001, 2048)])
def test_sandwich_many_rows(ops, dev, B, T, C, dt):
    _run(ops, dev, B, T, C, "rms", dt, ADA)
    _run(ops, dev, B, T, C, "layer", dt, AFFINE)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dt,vdt", [("f32", None), ("bf16", None), ("bf16", "f32")])
@pytest.mark.parametrize("C", [63, 255, 257, 1023, 1025, 2047, 2049, 4095, 4097, 8191, 8193])
def test_sandwich_unaligned_row_lengths(ops, dev, C, dt, vdt, kind):
    """Rows that do not start on 16 bytes: other threads per row from length to length."""
    _run(ops, dev, 3, 7, C, kind, dt, ADA if kind == "rms" else AFFINE, vdt=vdt)


@pytest.mark.parametrize("dt,C", [("f32", 8192), ("bf16", 16384)])
@pytest.mark.parametrize("vecs", [{"pw": "C", "w": "C"}, {"pw": "C", "pb": "C", "g": "BC", "w": "C", "b": "C", "sc": "BC"}])
def test_sandwich_rows_that_leave_little_room(ops, dev, dt, C, vecs):
    """Long rows whose coefficients leave room for one row or two in shared memory."""
    _run(ops, dev, 2, 170, C, "layer", dt, vecs)


def test_sandwich_large_mean(ops, dev):
    """A branch far from zero: the variance is of the centred values."""
    _run(ops, dev, 1, 64, 512, "layer", "f32", {}, mean=100.0)


@pytest.mark.parametrize("C", [512, 515])
def test_sandwich_in_place_and_last_block(ops, dev, C):
    import torch

    x, h, r, y = _run(ops, dev, 2, 30, C, "rms", "bf16", {"pw": "C", "g": "BC"})
    kw = dict(res_scale=0.5, norm="layer", eps=1e-6)
    r0, y0 = ops.sandwich_residual_norm(x, h, **kw)
    r1, none = ops.sandwich_residual_norm(x, h, next_norm=False, **kw)
    assert none is None and torch.equal(r0, r1)
    r2, y2 = ops.sandwich_residual_norm(x, h, inplace=True, **kw)
    assert r2 is x and torch.equal(x, r0) and torch.equal(y2, y0)


def test_sandwich_strided_rows_and_vectors(ops, dev):
    """x and h as column ranges of wider rows, the vectors as chunks of one."""
    import torch

    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 25, 3 * 320, generator=g).to(dev, torch.bfloat16)
    vec = torch.randn(2, 3 * 320, generator=g).to(dev, torch.bfloat16)
    gate, shift, scale = vec.chunk(3, -1)
    for off in (0, 320, 1):  # 1: not 16-byte aligned
        x, h = wide[..., off:off + 320], wide[..., 640 - off:960 - off]
        got = ops.sandwich_residual_norm(x, h, gate=gate, shift=shift, scale=scale)
        want = ops.sandwich_residual_norm(x.contiguous(), h.contiguous(), gate=gate.contiguous(),
                                          shift=shift.contiguous(), scale=scale.contiguous())
        for a, b in zip(got, want):
            assert (a.float() - b.float()).abs().max().item() <= 2.0 ** -5  # an ulp of the largest values


def test_sandwich_zero_rows_and_constant_rows(ops, dev):
    import torch

    x = torch.zeros(0, 64, device=dev)
    r, y = ops.sandwich_residual_norm(x, x)
    assert r.shape == y.shape == (0, 64)
    x = torch.full((3, 64), 2.0, device=dev)
    r, y = ops.sandwich_residual_norm(x, torch.zeros_like(x), norm="layer")  # no variance: eps alone
    assert torch.equal(r, x) and not y.any()
    r, y = ops.sandwich_residual_norm(x, torch.zeros_like(x), norm="rms")
    assert torch.equal(r, x) and torch.allclose(y, torch.ones_like(x), atol=1e-5)


def test_sandwich_nan_stays_in_its_row(ops, dev):
    import torch

    for C in (512, 331):
        x, h, r, y = _run(ops, dev, 2, 50, C, "layer", "bf16", AFFINE)
        h2 = h.clone()
        h2[0, 7, 3] = float("nan")
        r2, y2 = ops.sandwich_residual_norm(x, h2, res_scale=0.5)
        r1, y1 = ops.sandwich_residual_norm(x, h, res_scale=0.5)
        assert torch.isnan(r2[0, 7]).all() and torch.isnan(y2[0, 7]).all()
        r2[0, 7], y2[0, 7] = r1[0, 7], y1[0, 7]
        assert torch.equal(r2, r1) and torch.equal(y2, y1)


def test_sandwich_other_stream_and_graph(ops, dev):
    import torch

    x, h, _, _ = _run(ops, dev, 2, 300, 1024, "rms", "bf16", ADA)
    want = ops.sandwich_residual_norm(x, h)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            kept = ops.sandwich_residual_norm(x, h)
        g.replay()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_sandwich_refusals(pkg, ops, dev):
    import torch

    x = torch.zeros(2, 5, 64, device=dev)
    bad = [
        (dict(h=x[:, :4]), "shape"), (dict(h=x.half()), "dtype"), (dict(gate=torch.zeros(3, 64, device=dev)), "batch"),
        (dict(weight=torch.zeros(63, device=dev)), "last dim"), (dict(eps=-1.0), "eps"),
        (dict(next_norm=False, weight=torch.zeros(64, device=dev)), "need y"),
        (dict(x=x.int(), h=x.int()), "F32/F16/BF16"),
        (dict(x=torch.zeros(1, 30000, device=dev), h=torch.zeros(1, 30000, device=dev)), "exceeds"),
        (dict(h=torch.zeros(2, 64, 5, device=dev).transpose(1, 2)), "contiguous"),
    ]
    for kw, match in bad:
        with pytest.raises(pkg._lib.L3dError, match=match):
            ops.sandwich_residual_norm(**({"x": x, "h": x} | kw))
    with pytest.raises(KeyError):
        ops.sandwich_residual_norm(x, x, norm="batch")
    with pytest.raises(ValueError, match="CUDA"):
        ops.sandwich_residual_norm(x.cpu(), x)


def test_checked_calls_pass_on_an_idle_status_word(pkg, ops, dev):
    """check=True after calls that finish: no error, the same bits, the word still 0."""
    import torch

    x = torch.randn(3, 40, 512, device=dev).to(torch.bfloat16)
    r, y = ops.sandwich_residual_norm(x, x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.sandwich_residual_norm(x, x, check=True)
        q = x.view(3, 40, 8, 64).transpose(1, 2)
        ops.shared_prefix_attention(q, q[0], q[0], check=True)
        ad = ops.LoraAdapters([torch.ones(4, 512, device=dev)], [torch.ones(64, 4, device=dev)])
        w = torch.zeros(64, 512, device=dev, dtype=torch.bfloat16)
        ops.lora_linear(x, w, ad, torch.zeros(3, device=dev, dtype=torch.int32), check=True)
    assert torch.equal(got[0], r) and torch.equal(got[1], y)
    assert ops.kernel_status(dev) == 0


@pytest.mark.parametrize("dt,u", [("f32", 2.0 ** -24), ("bf16", 2.0 ** -8), ("f16", 2.0 ** -11)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("T,C", [(3, 64), (400, 256), (33, 1024), (170, 2048), (5, 8192), (7, 77), (9, 2047), (2, 20001)])
def test_sandwich_is_as_near_as_its_output_type(ops, dev, T, C, kind, dt, u):
    """Within the rounding of the stored value and 1e-5 of the terms that are added
    up: f32 statistics of up to 20001 elements in sums of several parts, some 20
    roundings, once each for r and for y's own norm of it."""
    r = rng(77 + T * C)
    names = {"pw": 1.0, "pb": 0.0, "g": 1.0, "w": 1.0, "b": 0.0, "sh": 0.0, "sc": 0.0}
    x, xv = to_dev(r.standard_normal((2, T, C)), dt, dev)
    h, hv = to_dev(3 * r.standard_normal((2, T, C)) + 0.3, dt, dev)
    t, f = {}, {}
    for name, mean in names.items():
        t[name], v = to_dev(mean + 0.2 * r.standard_normal((2, C) if name in ("g", "sh", "sc") else (C,)), dt, dev)
        f[name] = v.astype(np.float64)
    ro, yo = ops.sandwich_residual_norm(x, h, post_weight=t["pw"], post_bias=t["pb"], gate=t["g"], res_scale=0.75,
                                        weight=t["w"], bias=t["b"], shift=t["sh"], scale=t["sc"], norm=kind,
                                        eps=1e-5, post_eps=1e-6)
    xv, hv = xv.astype(np.float64), hv.astype(np.float64)
    rr, yr = _ref(kind, xv, hv, f["pw"], f["pb"], f["g"], 0.75, f["w"], f["b"], f["sh"], f["sc"], 1e-6, 1e-5)
    per = lambda n: f[n].reshape(2, 1, C)  # noqa: E731
    nrm = np.abs(_norm(kind, hv, None, None, 1e-6))
    terms = 0.75 * np.abs(xv) + np.abs(per("g")) * (nrm * np.abs(f["pw"]) + np.abs(f["pb"]))
    v = rr - rr.mean(-1, keepdims=True) if kind == "layer" else rr
    inv = 1 / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-5)
    terms_y = (1 + np.abs(per("sc"))) * (np.abs(f["w"]) * inv * (terms + terms.mean(-1, keepdims=True)) + np.abs(f["b"])) \
        + np.abs(per("sh"))
    for got, want, mag in ((ro, rr, terms), (yo, yr, terms_y)):
        err = np.abs(got.double().cpu().numpy() - want)
        bound = u * np.abs(want) + 1e-5 * mag + (2.0 ** -25 if dt == "f16" else 0.0)
        assert (err <= bound).all(), (err / bound).max()
