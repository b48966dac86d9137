"""GPU: paged attention where a head's keys are divided between warps, by each of the ways their parts are joined
(the bounds of test_gpu_paged).  Which way a call takes follows from its sizes; each test says which it is after,
and works it out from them."""
import pytest

from conftest import rng
from test_gpu_paged import _run_attention

pytestmark = pytest.mark.gpu


def _way(dev, lens, N, Hq, Hkv, D, size, room):
    """"alone", "ends", or the joining kernel's warps for a row; and the parts that the longest head comes in."""
    import torch

    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    B, R, kt = len(lens), N * Hq // Hkv, 32 if D == 64 else 16
    row_tiles = 1 if R <= 8 else -(-R // 16)
    heads = B * Hkv * row_tiles
    longest = (-(-max(lens) // size) + (9000 // size if room else 0)) * size
    if heads <= sms and longest <= (4 + heads // 24) * 12 * kt:
        return "alone", 12
    full = -(-longest // kt)
    warps = 12 * min(max(heads * full, 1), sms)
    real = max(-(-sum(-(-n // kt) for n in lens) * Hkv * row_tiles // warps), 1)
    parts = -(-max(lens) // kt) / real
    if heads > warps:
        return "ends", parts
    many = full // max(-(-heads * full // warps), 1)
    return 1 if many <= 8 else 8 if B * Hkv * R > 2 * sms else 16 if many <= 160 else 32, parts


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("way,lens,N,Hq,Hkv,size,room", [
    (1, [4096, 100, 3000, 4000] * 16, 1, 16, 4, 16, False),
    (1, [600, 555, 90, 17] * 8, 16, 8, 2, 16, False),            # 64 rows a head, four row tiles
    (8, [4101, 4000, 3500, 1, 0, 4100, 2000, 3, 4099, 77, 4101, 4096], 4, 12, 12, 16, False),
    (8, [2500, 1400], 16, 16, 2, 32, True),                      # 128 rows a head, eight row tiles
    (8, [900, 0, 333], 20, 12, 4, 48, True),                     # 60 rows, the last row tile of twelve
    (16, [2500, 1400], 7, 5, 1, 16, False),                      # 35 rows, three row tiles
    (16, [2400, 70, 900], 1, 8, 2, 1, False),
    (32, [20000], 2, 16, 2, 256, False),
    (32, [30000, 9], 9, 4, 1, 64, False),                        # 36 rows
])
def test_joined_by_rows(ops, dev, way, lens, N, Hq, Hkv, size, room, D, dt):
    got, parts = _way(dev, lens, N, Hq, Hkv, D, size, room)
    assert got == way and parts > 2, (got, parts)
    _run_attention(ops, dev, lens, N, Hq, Hkv, D, size, dt, wide=room)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,longest,N,Hq,Hkv", [
    (450, 350, 1, 8, 4),      # two rows a head
    (450, 350, 2, 32, 4),     # sixteen
    (160, 500, 7, 20, 4),     # 35: three row tiles
    (100, 400, 16, 24, 3),    # 128: eight row tiles
])
def test_joined_at_the_ends_of_stretches(ops, dev, B, longest, N, Hq, Hkv, D, dt):
    lens = rng(B + N).integers(0, longest, B).tolist()
    lens[:3], lens[-2:], lens[B // 2] = [0, 1, longest], [longest, 0], 6000
    got, parts = _way(dev, lens, N, Hq, Hkv, D, 16, False)
    assert got == "ends" and parts > 2, (got, parts)
    _run_attention(ops, dev, lens, N, Hq, Hkv, D, 16, dt)
