"""GPU: small probabilities in f16, in paged attention and in the attention of packed sequences, against softmax in
f64 on the same inputs.

Bounds as in test_gpu_paged and test_gpu_cross_attention, but for what f16 loses of small probabilities.  They are
held with the largest one of a stretch of keys at 2^7 or more (2^15 at most, so that 65504 is not reached) while f16
goes down in steps of 2^-24: a pair of parts is off by at most 2^-24 there, 2^-31 of the row's largest probability a
key; a single part by half of that, 2^-32."""
import pytest

from conftest import rng
from test_gpu_paged import U, _ints

pytestmark = pytest.mark.gpu


def _few_large(r, n, D, gap, dev):
    """q and n keys of which every 256th scores some `gap` nats above the others (0), with V = 0; the others' V are
    1 to 2."""
    import torch

    q, k = torch.zeros(D, device=dev), torch.zeros(n, D, device=dev)
    q[0], k[::256, 0] = 8.0, gap * D ** 0.5 / 8.0
    v = 1.0 + torch.from_numpy(r.random((n, D))).to(dev)
    v[::256] = 0
    return q.half(), k.half(), v.half()


GAPS = [6.0, 8.3, 9.9, 11.1, 12.0, 12.7, 13.3, 13.9, 14.6]


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", ["pages", "pages alone", "packed"])
def test_small_probabilities_of_two_parts(ops, dev, form, D, gap):
    """Thousands of keys that weigh little each keep their weight beside a few that weigh much."""
    import torch

    B, H, n = (64, 4, 4096) if form != "pages alone" else (4, 4, 700)
    q1, k1, v1 = _few_large(rng(D), n, D, gap, dev)
    q = q1.expand(B, H, D).contiguous()
    if form == "packed":
        k, v = (t[:, None].expand(n, H, D).repeat(B, 1, 1) for t in (k1, v1))
        out = ops.cross_attention(q, k, v, torch.arange(B + 1, dtype=torch.int32, device=dev) * n, check=True)
    else:
        size = 4
        kp, vp = (t.view(n // size, size, 1, D).expand(-1, -1, H, -1) for t in (k1, v1))
        table = torch.arange(n // size, dtype=torch.int32, device=dev).expand(B, -1).contiguous()
        out = ops.paged_attention(q, kp, vp, table, _ints([n] * B, dev), check=True)
    p = torch.softmax((k1.double() @ q1.double()) * D ** -0.5, 0)
    want = p @ v1.double()
    bound = U["f16"] * want + (1.4e-4 + 2.0 ** -16 + 1e-5) * want + n * 2.0 ** -31 * p.max() * 2 + 2.0 ** -25
    err = (out.double() - want).abs()
    assert (err <= bound).all(), f"worst ratio {(err / bound).max().item():.2f}"


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,n", [(40, 4096), (128, 1024)])
def test_small_probabilities_of_one_part(ops, dev, rows, n, D, gap):
    """Many rows over packed keys: each probability rounded once, to 2^-11 of itself or 2^-32 of the row's largest."""
    import torch

    B, H = 80, 4
    q1, k1, v1 = _few_large(rng(D), n, D, gap, dev)
    q = q1.expand(B * rows, H, D).contiguous()
    k, v = (t[:, None].expand(n, H, D).repeat(B, 1, 1) for t in (k1, v1))
    out = ops.cross_attention(q, k, v, torch.arange(B + 1, dtype=torch.int32, device=dev) * n, check=True)
    p = torch.softmax((k1.double() @ q1.double()) * D ** -0.5, 0)
    want = p @ v1.double()
    bound = (2 * U["f16"] + 4e-4) * want + n * 2.0 ** -32 * p.max() * 2 + 2.0 ** -25
    err = (out.double() - want).abs()
    assert (err <= bound).all(), f"worst ratio {(err / bound).max().item():.2f}"
