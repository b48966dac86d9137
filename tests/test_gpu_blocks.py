"""GPU parity of the block stacks (fused ops + cuBLAS GEMMs + attention, both
torch SDPA and l3d_attention) against plain torch f32 restatements of the
reference blocks at reduced depth/size.

Stacks compound bf16 rounding across blocks, so the comparison is normwise:
relative L2 error of the stack output (and of the residual-stream update)
within 2e-2, the bf16 tolerance of the parity contract applied to the whole
block rather than to one op.
"""
import pytest

pytestmark = pytest.mark.gpu


def rel_l2(a, b):
    a, b = a.float(), b.float()
    return float((a - b).norm() / b.norm())


@pytest.fixture(params=["sdpa", "l3d"])
def attn(request, pkg):
    """The stacks' bf16 attention core: torch SDPA, or l3d_attention."""
    from candle3d_b200 import blocks

    blocks.set_attention(request.param)
    yield request.param
    blocks.set_attention("sdpa")


@pytest.mark.parametrize("fused_mlp", [False, True])
def test_vggt_stack_matches_reference(pkg, dev, attn, fused_mlp, monkeypatch):
    import torch

    from candle3d_b200 import blocks

    # fused_mlp: fc1 + GELU-erf as one tcgen05 GEMM at any size (normally from
    # 8192 rows).
    monkeypatch.setattr(blocks, "FUSED_MLP_MIN_ROWS", 0 if fused_mlp else 1 << 62)

    # LayerScale 1.0 instead of the 0.01 init: with 0.01 the per-block update
    # is far below one bf16 ulp of the residual stream and rounds away (in
    # Candle's bf16 path as well), leaving nothing to compare.
    agg = blocks.VggtAggregator(depth=2, device=dev, ls_init=1.0)
    B, S, ph, pw, special = 1, 2, 9, 9, 5
    N = special + ph * pw
    fpos = blocks.VggtAggregator.positions(B, S, ph, pw, special, dev)
    gpos = fpos.reshape(B, S * N, 2)
    g = torch.Generator().manual_seed(1)
    tok = torch.randn(B * S, N, 1024, generator=g).to(dev, torch.bfloat16)
    ref = blocks.vggt_reference(agg, tok, fpos, gpos, S)
    out = agg.forward(tok.clone(), fpos, gpos, S)
    assert rel_l2(out - tok, ref - tok.float()) < 2e-2
    assert rel_l2(out, ref) < 2e-2


def test_triposg_stack_matches_reference(pkg, dev, attn):
    import torch

    from candle3d_b200 import blocks

    m = blocks.TripoSgDit(layers=5, device=dev)
    g = torch.Generator().manual_seed(2)
    lat = torch.randn(2, 64, 64, generator=g).to(dev, torch.bfloat16)
    cond = torch.randn(2, 37, 1024, generator=g).to(dev, torch.bfloat16)
    cond[0].zero_()  # CFG batch [uncond (zeros), cond]
    t = torch.tensor([370.0], device=dev)
    out = m.forward(lat, t, cond)
    ref = blocks.triposg_reference(m, lat, t, cond)
    assert out.shape == (2, 64, 64)
    assert rel_l2(out, ref) < 2e-2


def test_trellis_slat_stack_matches_reference(pkg, ops, dev, attn):
    import torch
    import torch.nn.functional as F

    from candle3d_b200 import blocks

    m = blocks.Trellis2Slat(blocks=2, device=dev)
    g = torch.Generator().manual_seed(3)
    occ = torch.rand(16, 16, 16, generator=g) < 0.12
    coords = torch.nonzero(occ).to(torch.int32).to(dev)
    N = coords.shape[0]
    feats = torch.randn(N, 32, generator=g).to(dev, torch.bfloat16)
    cond = torch.randn(1, 40, 1024, generator=g).to(dev, torch.bfloat16)
    t = torch.tensor([650.0], device=dev)
    out = m.forward(feats, coords, t, cond)

    # torch f32 restatement of Trellis2SparseBlock / SLAT forward with the
    # dequantised weights (crate/runtime/trellis2_blocks.rs:609-646).
    f = lambda a: a.float()  # noqa: E731

    def lin(q, x):
        w = ops.dequantize(q.blocks, "q8_0", q.n, q.k)
        return F.linear(x, w, q.bias)

    C, H, D = m.C, m.H, m.D
    half = 128
    freqs = torch.exp(-torch.log(torch.tensor(10000.0)) * torch.arange(half) / half).to(dev)
    arg = t.float() * freqs
    tab = torch.cat([torch.cos(arg), torch.sin(arg)]).view(1, 256)
    th = F.linear(F.silu(F.linear(tab, f(m.t_fc1[0]), f(m.t_fc1[1]))), f(m.t_fc2[0]), f(m.t_fc2[1]))
    temb = F.linear(F.silu(th), f(m.ada[0]), f(m.ada[1]))
    cs, sn = ops.Trellis2Rope3d(D).cos_sin(coords)

    def qknorm(x, gamma):
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-12) * gamma * D ** 0.5

    def rope(x):
        z = torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous())
        rot = torch.polar(torch.ones_like(cs), torch.atan2(sn, cs))
        return torch.view_as_real(z * rot[None, :, None, :]).reshape(x.shape)

    x = F.linear(f(feats), f(m.input_layer[0]), f(m.input_layer[1])).view(1, N, C)
    for p in m.blocks:
        mv = f(p["modulation"]).unsqueeze(0) + temb
        sh1, sc1, g1, sh2, sc2, g2 = [c.unsqueeze(1) for c in mv.chunk(6, -1)]
        h = F.layer_norm(x, (C,), eps=1e-6) * (1 + sc1) + sh1
        qkv = lin(p["to_qkv"], h).view(1, N, 3, H, D)
        q = rope(qknorm(qkv[:, :, 0], p["qg"]))
        k = rope(qknorm(qkv[:, :, 1], p["kg"]))
        a = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), qkv[:, :, 2].transpose(1, 2))
        x = x + g1 * lin(p["to_out"], a.transpose(1, 2).reshape(1, N, C))
        h = F.layer_norm(x, (C,), f(p["n2w"]), f(p["n2b"]), 1e-6)
        cq = qknorm(lin(p["c_q"], h).view(1, N, H, D), p["cqg"])
        kv = lin(p["c_kv"], f(cond)).view(1, -1, 2, H, D)
        ck = qknorm(kv[:, :, 0], p["ckg"])
        ca = F.scaled_dot_product_attention(cq.transpose(1, 2), ck.transpose(1, 2), kv[:, :, 1].transpose(1, 2))
        x = x + lin(p["c_out"], ca.transpose(1, 2).reshape(1, N, C))
        h = F.layer_norm(x, (C,), eps=1e-6) * (1 + sc2) + sh2
        x = x + g2 * lin(p["mlp2"], F.gelu(lin(p["mlp0"], h), approximate="tanh"))
    ref = F.linear(F.layer_norm(x, (C,), eps=1e-5).view(N, C), f(m.out_layer[0]), f(m.out_layer[1]))
    assert out.shape == (N, 32)
    assert rel_l2(out, ref) < 2e-2


def _shared_context(dev, P, B, L):
    import torch

    from candle3d_b200 import blocks

    m = blocks.SharedContextBlocks(device=dev)
    g = torch.Generator().manual_seed(P)
    tokens = torch.randn(P, m.C, generator=g).to(dev, torch.bfloat16)
    x = torch.randn(B, L, m.C, generator=g).to(dev, torch.bfloat16)
    ids = torch.tensor([b % 4 if b % 4 < 3 else -1 for b in range(B)], dtype=torch.int32, device=dev)
    cache = m.new_cache(B, L + 9)
    for k, v in cache:  # what lies past a request's own tokens must not matter
        k.fill_(float("nan"))
        v.fill_(float("nan"))
    return m, x, ids, m.encode_context(tokens), cache, blocks.shared_context_reference(m, x, tokens, ids)


@pytest.mark.parametrize("P,steps,B", [(200, (5, 1, 1, 3), 4), (64, (1, 1), 1), (1000, (33, 1), 7)])
def test_shared_context_blocks_match_reference(pkg, dev, P, steps, B):
    """Requests with adapters of their own around one context, their tokens in
    steps through the caches, against whole sequences at once in f64."""
    import torch

    m, x, ids, context, cache, ref = _shared_context(dev, P, B, sum(steps))
    outs, at = [], 0
    for n in steps:
        start = torch.full((B,), at, dtype=torch.int32, device=dev)
        outs.append(m.forward(x[:, at:at + n].contiguous(), context, cache, start, ids))
        at += n
    assert rel_l2(torch.cat(outs, 1), ref) < 2e-2


def test_shared_context_blocks_ragged_requests(pkg, dev):
    """Requests that join with different numbers of tokens, then step together."""
    import torch

    have = [1, 17, 4, 30, 8]
    m, x, ids, context, cache, ref = _shared_context(dev, 300, len(have), 32)
    for b, n in enumerate(have):
        own = [(k[b:b + 1], v[b:b + 1]) for k, v in cache]
        y = m.forward(x[b:b + 1, :n].contiguous(), context, own,
                      torch.zeros(1, dtype=torch.int32, device=dev), ids[b:b + 1])
        assert rel_l2(y, ref[b:b + 1, :n]) < 2e-2
    start = torch.tensor(have, dtype=torch.int32, device=dev)
    for _ in range(2):
        rows = torch.arange(len(have), device=dev)
        y = m.forward(x[rows, start.long()].unsqueeze(1), context, cache, start, ids)
        assert rel_l2(y[:, 0], ref[rows, start.long()]) < 2e-2
        start = start + 1


@pytest.mark.parametrize("N", [1, 3])
def test_shared_context_blocks_past_a_cache(pkg, dev, N):
    """A request whose tokens do not fit its cache, or that claims to hold fewer than
    none, comes out NaN; the others keep their bits and their caches."""
    import torch

    B, have = 4, 6
    m, x, ids, context, cache, _ = _shared_context(dev, 100, B, 9)
    room = cache[0][0].shape[2]
    m.forward(x[:, :have].contiguous(), context, cache, torch.zeros(B, dtype=torch.int32, device=dev), ids)
    step, start = x[:, have:have + N].contiguous(), torch.full((B,), have, dtype=torch.int32, device=dev)
    copy = [(k.clone(), v.clone()) for k, v in cache]
    want = m.forward(step, context, copy, start, ids)
    bad = start.clone()
    bad[1], bad[3] = room - N + 1, -1
    got = m.forward(step, context, cache, bad, ids)
    good = [0, 2]
    assert torch.isnan(got[1]).all() and torch.isnan(got[3]).all() and torch.equal(got[good], want[good])
    for (k, v), (k2, v2) in zip(cache, copy):
        assert torch.equal(k[good][:, :, :have + N], k2[good][:, :, :have + N])
        assert torch.equal(v[good][:, :, :have + N], v2[good][:, :, :have + N])
    with pytest.raises(ValueError, match="do not fit"):
        m.forward(torch.zeros(B, room + 1, m.C, device=dev, dtype=x.dtype), context, cache, start, ids)
