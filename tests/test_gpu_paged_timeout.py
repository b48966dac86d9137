"""GPU: a wait that runs out in the kernel of l3d_paged_attention leaves an error behind, and nothing else: the
kernel that joins the parts, launched behind it either way, stays within the tensors whatever the workspace held."""
import pytest

from test_gpu_paged import _ints, _pages, _rand
from conftest import rng

pytestmark = pytest.mark.gpu

FORMS = {
    "alone": dict(lens=[40, 7, 0], N=1, Hq=4, Hkv=2, room=0),       # a block for each head: no workspace
    "line": dict(lens=[900, 3000], N=1, Hq=4, Hkv=2, room=9000),    # every row looked at by the joining kernel
    "ends": dict(lens=[70, 300, 0, 5] * 75, N=2, Hq=24, Hkv=8, room=0),  # more heads than warps: only the stretches' ends
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fill", [0x7F, 0xFF, 0x01])
def test_paged_attention_timeout_is_contained(pkg, ops, dev, form, fill):
    import torch

    lens, N, Hq, Hkv, room = FORMS[form].values()
    D, size, B = 64, 16, len(lens)
    r = rng(B)
    kp, vp, table, _ = _pages(r, lens, size, Hkv, D, "bf16", dev)
    if room:
        table = torch.cat([table, torch.full((B, room // size), -1, dtype=torch.int32, device=dev)], 1)
    q, held = _rand(r, (B, N, Hq, D), "bf16", dev), _ints(lens, dev)
    good = ops.paged_attention(q, kp, vp, table, held, check=True)
    L = pkg._lib
    lib = L.lib()
    need = lib.l3d_paged_attention_workspace_size(B, Hq, Hkv, N, table.shape[1] * size, D)
    assert (need == 0) == (form == "alone")
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    assert (B * Hkv > sms * 12) == (form == "ends")
    ws = torch.full((max(need, 256),), fill, dtype=torch.uint8, device=dev)
    store = torch.full((3, *q.shape), 7.0, dtype=q.dtype, device=dev)  # the output between two guards
    stream = torch.cuda.current_stream(dev).cuda_stream

    def run(ms):
        return lib.l3d_paged_attention_selftest_timeout(*(L.packed(t) for t in (q, kp, vp, table, held)), D ** -0.5,
                                                        L.packed(store[1]), ws.data_ptr(), need, ms, stream)
    assert run(0) == 4 and run(2001) == 4
    assert run(30) == 0, lib.l3d_last_error()
    torch.cuda.synchronize()
    assert ops.kernel_status(dev) == 5
    assert (store[0] == 7).all() and (store[2] == 7).all()
    if form != "line":  # (there the joining kernel weighs what the workspace held)
        have = held > 0
        assert (store[1][have] == 7).all()
    assert ops.kernel_status(dev) == 0
    assert torch.equal(ops.paged_attention(q, kp, vp, table, held, check=True), good)
