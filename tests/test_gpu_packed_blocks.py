"""GPU: batches of different lengths through the block stacks (packed encoder tokens,
packed scenes, requests over a paged cache), against each element by itself.

The stacks round to bf16 after every op; as in test_gpu_blocks.py the comparison is
normwise, relative L2 error within 2e-2."""
import pytest

from test_gpu_blocks import rel_l2

pytestmark = pytest.mark.gpu


def _offsets(lens, dev):
    import numpy as np
    import torch

    return torch.tensor(np.cumsum([0, *lens]), dtype=torch.int32, device=dev)


def test_triposg_packed_encoder_tokens(pkg, dev):
    """Objects whose images gave different numbers of tokens, in one batch."""
    import torch

    from candle3d_b200 import blocks

    m = blocks.TripoSgDit(layers=3, C=512, H=4, ff=1024, device=dev)
    g = torch.Generator().manual_seed(5)
    lens = [77, 300, 130]
    lat = torch.randn(3, 200, 64, generator=g).to(dev, torch.bfloat16)
    cond = torch.randn(sum(lens), 1024, generator=g).to(dev, torch.bfloat16)
    t = torch.tensor(0.4, device=dev)
    out = m.forward(lat, t, cond, cond_offsets=_offsets(lens, dev))
    for b, c in enumerate(cond.split(lens)):
        ref = blocks.triposg_reference(m, lat[b:b + 1], t, c[None])
        alone = m.forward(lat[b:b + 1], t, c[None])
        assert rel_l2(out[b:b + 1], ref) < 2e-2
        # The packed form is as near the f32 one as the batch of one is, within the rounding of both.
        assert rel_l2(out[b:b + 1], ref) < 1.5 * rel_l2(alone, ref) + 2e-3
    with pytest.raises(ValueError, match="offsets"):
        m.forward(lat, t, cond, cond_offsets=_offsets(lens[:2], dev))
    with pytest.raises(ValueError, match="offsets"):
        m.forward(lat, t, cond[None], cond_offsets=_offsets(lens, dev))


def test_trellis_packed_scenes(pkg, dev):
    """Scenes of different sizes with images of their own, in one pass."""
    import torch

    from candle3d_b200 import blocks

    m = blocks.Trellis2Slat(blocks=2, C=512, H=4, mlp=1024, device=dev)
    g = torch.Generator().manual_seed(6)
    rows, lens = [500, 40, 900], [130, 257, 77]
    feats = torch.randn(sum(rows), 32, generator=g).to(dev, torch.bfloat16)
    coords = torch.randint(0, 64, (sum(rows), 3), generator=g, dtype=torch.int32).to(dev)
    cond = torch.randn(sum(lens), 1024, generator=g).to(dev, torch.bfloat16)
    t = torch.tensor(0.7, device=dev)
    out = m.forward(feats, coords, t, cond, scene_offsets=_offsets(rows, dev), cond_offsets=_offsets(lens, dev))
    for got, f, c, e in zip(out.split(rows), feats.split(rows), coords.split(rows), cond.split(lens)):
        assert rel_l2(got, m.forward(f.contiguous(), c.contiguous(), t, e[None])) < 2e-2
    for bad in (dict(scene_offsets=_offsets(rows, dev)), dict(cond_offsets=_offsets(lens, dev))):
        with pytest.raises(ValueError, match="packed scenes"):
            m.forward(feats, coords, t, cond, **bad)


def _requests(dev, lens, states, size=16, spare=3, seed=0):
    """A model, tokens of len(lens) requests, their encoder states, a cache with room for them."""
    import torch

    from candle3d_b200 import blocks

    m = blocks.PagedRequestBlocks(device=dev)
    g = torch.Generator().manual_seed(seed)
    B, L = len(lens), max(lens)
    x = torch.randn(B, L, m.C, generator=g).to(dev, torch.bfloat16)
    st = torch.randn(sum(states), 1024, generator=g).to(dev, torch.bfloat16)
    pos = torch.randint(0, 400, (B, L, 3), generator=g, dtype=torch.int32).to(dev)
    ids = torch.tensor([i % 4 - 1 for i in range(B)], dtype=torch.int32, device=dev)
    need = [-(-n // size) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)])
    cache = m.new_pages(sum(need) + spare, size)
    refs = [blocks.paged_request_reference(m, x[b, :lens[b]], s, pos[b, :lens[b]], int(ids[b]))
            for b, s in enumerate(st.split(states))]
    return m, x, m.encode_states(st), _offsets(states, dev), cache, table.to(dev), pos, ids, refs


@pytest.mark.parametrize("steps,states", [((5, 1, 1, 3), [300, 77, 130, 1]), ((1, 1, 1), [1029]), ((33, 1, 2), [64, 200, 5])])
def test_paged_requests_in_steps(pkg, dev, steps, states):
    """Tokens in steps through the pages, encoder states of different lengths, adapters of their own."""
    import torch

    B, L = len(states), sum(steps)
    m, x, kv, so, cache, table, pos, ids, refs = _requests(dev, [L] * B, states)
    outs, at = [], 0
    for n in steps:
        held = torch.full((B,), at, dtype=torch.int32, device=dev)
        outs.append(m.forward(x[:, at:at + n].contiguous(), kv, so, cache, table, held, ids, pos[:, at:at + n]))
        at += n
    assert rel_l2(torch.cat(outs, 1), torch.stack(refs)) < 2e-2


def test_paged_requests_ragged(pkg, dev):
    """Requests that hold different numbers of tokens step together, one captured step for all lengths."""
    import torch

    lens, states = [3, 40, 17, 1], [50, 257, 4, 130]
    m, x, kv, so, cache, table, pos, ids, refs = _requests(dev, [n + 3 for n in lens], states, seed=3)
    for b, n in enumerate(lens):  # each request's first tokens by themselves
        first = torch.zeros(1, dtype=torch.int32, device=dev)
        mine = [(k[so[b]:so[b + 1]], v[so[b]:so[b + 1]]) for k, v in kv]
        y = m.forward(x[b:b + 1, :n].contiguous(), mine, _offsets([states[b]], dev), cache, table[b:b + 1], first,
                      ids[b:b + 1], pos[b:b + 1, :n])
        assert rel_l2(y[0], refs[b][:n]) < 2e-2
    held = torch.tensor(lens, dtype=torch.int32, device=dev)
    rows = torch.arange(len(lens), device=dev)
    xs, ps = x[rows, held.long()].unsqueeze(1).clone(), pos[rows, held.long()].unsqueeze(1).clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # warm-up, of a step that is repeated below with the same result
        m.forward(xs, kv, so, cache, table, held, ids, ps)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.forward(xs, kv, so, cache, table, held, ids, ps)
    for _ in range(3):
        xs.copy_(x[rows, held.long()].unsqueeze(1))
        ps.copy_(pos[rows, held.long()].unsqueeze(1))
        graph.replay()
        for b in range(len(lens)):
            assert rel_l2(y[b, 0], refs[b][int(held[b])]) < 2e-2
        held += 1


def test_paged_requests_past_their_pages(pkg, dev):
    """A request without room comes out NaN; the others and their pages keep their bits."""
    import torch

    m, x, kv, so, cache, table, pos, ids, _ = _requests(dev, [32, 32, 32], [40, 30, 20], seed=9)
    held = torch.full((3,), 30, dtype=torch.int32, device=dev)
    copy = [(k.clone(), v.clone()) for k, v in cache]
    want = m.forward(x[:, :2].contiguous(), kv, so, copy, table, held, ids, pos[:, :2])
    bad = held.clone()
    bad[1] = 31  # its second token has no page
    got = m.forward(x[:, :2].contiguous(), kv, so, cache, table, bad, ids, pos[:, :2])
    assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2]], want[[0, 2]])
    mine = set(table[1].tolist())
    for (k, v), (k2, v2) in zip(cache, copy):
        other = [i for i in range(k.shape[0]) if i not in mine]
        assert torch.equal(k[other], k2[other]) and torch.equal(v[other], v2[other])
