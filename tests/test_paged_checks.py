"""CPU: the entries of a paged cache refuse invalid requests on the host, before any launch."""
import math

import numpy as np
import pytest

from test_serving_checks import E_ALIGN, E_DTYPE, E_NULL, E_SHAPE, E_UNSUPPORTED, E_WORKSPACE, _refused, _zeros


def _append_args(**over):
    T, Hq, Hkv, D, B = 6, 4, 2, 64, 3
    a = dict(q=_zeros(T, Hq, D), k=_zeros(T, Hkv, D), v=_zeros(T, Hkv, D), q_weight=_zeros(D), k_weight=_zeros(D),
             eps=1e-6, freqs=_zeros(32, 2, dtype="float32"), axes=_zeros(32, dtype="int32"), half=32,
             positions=_zeros(T, 2, dtype="int32"), table=_zeros(B, 5, dtype="int32"), held=_zeros(B, dtype="int32"),
             offsets=_zeros(B + 1, dtype="int32"), q_out=_zeros(T, Hq, D), k_pages=_zeros(7, 16, Hkv, D),
             v_pages=_zeros(7, 16, Hkv, D))
    assert not set(over) - set(a)
    return [*(a | over).values(), None]


@pytest.mark.parametrize("over,code,word", [
    (dict(q=None), E_NULL, "required"),
    (dict(table=None), E_NULL, "required"),
    (dict(held=None), E_NULL, "required"),
    (dict(k_weight=None), E_NULL, "together"),
    (dict(axes=None), E_NULL, "together"),
    (dict(freqs=None, axes=None), E_SHAPE, "positions need freqs"),
    (dict(q=_zeros(6, 4, 64, dtype="float32")), E_DTYPE, "BF16"),
    (dict(k_pages=_zeros(7, 16, 2, 64, dtype="float16")), E_DTYPE, "F16"),
    (dict(v=_zeros(6, 128)), E_SHAPE, "[T, H, D]"),
    (dict(k_pages=_zeros(7, 32, 64)), E_SHAPE, "[pages, size, H, D]"),
    (dict(k=_zeros(6, 64, 2).transpose(1, 2)), E_ALIGN, "contiguous"),
    (dict(q=_zeros(6, 4, 32), q_out=_zeros(6, 4, 32)), E_UNSUPPORTED, "64 or 128"),
    (dict(q_out=_zeros(6, 5, 64)), E_SHAPE, "q_out"),
    (dict(v=_zeros(6, 3, 64)), E_SHAPE, "k and v"),
    (dict(k=_zeros(5, 2, 64), v=_zeros(5, 2, 64)), E_SHAPE, "k and v"),
    (dict(v_pages=_zeros(7, 17, 2, 64)), E_SHAPE, "k_pages and v_pages"),
    (dict(k_pages=_zeros(7, 16, 3, 64), v_pages=_zeros(7, 16, 3, 64)), E_SHAPE, "k_pages and v_pages"),
    (dict(k_pages=_zeros(7, 0, 2, 64), v_pages=_zeros(7, 0, 2, 64)), E_UNSUPPORTED, "pages of no tokens"),
    (dict(table=_zeros(3, 5, dtype="int64")), E_DTYPE, "table"),
    (dict(table=_zeros(15, dtype="int32")), E_SHAPE, "table"),
    (dict(table=_zeros(5, 3, dtype="int32").t()), E_SHAPE, "contiguous rows"),
    (dict(held=_zeros(4, dtype="int32")), E_SHAPE, "held"),
    (dict(held=_zeros(3, dtype="float32")), E_SHAPE, "held"),
    (dict(offsets=_zeros(3, dtype="int32")), E_SHAPE, "offsets"),
    (dict(offsets=_zeros(8, dtype="int32")[::2]), E_SHAPE, "offsets"),
    (dict(offsets=None, q=_zeros(7, 4, 64), k=_zeros(7, 2, 64), v=_zeros(7, 2, 64), q_out=_zeros(7, 4, 64),
          positions=None), E_SHAPE, "divide evenly"),
    (dict(eps=-1.0), E_UNSUPPORTED, "eps"),
    (dict(eps=math.nan), E_UNSUPPORTED, "eps"),
    (dict(freqs=_zeros(32, 2)), E_DTYPE, "freqs"),
    (dict(freqs=_zeros(33, 2, dtype="float32"), axes=_zeros(33, dtype="int32")), E_SHAPE, "D / 2 pairs"),
    (dict(axes=_zeros(31, dtype="int32")), E_SHAPE, "pairs"),
    (dict(half=12), E_UNSUPPORTED, "half"),
    (dict(half=24), E_UNSUPPORTED, "half"),
    (dict(half=-8), E_UNSUPPORTED, "half"),
    (dict(positions=_zeros(6, 2, dtype="float32")), E_DTYPE, "positions"),
    (dict(positions=_zeros(5, 2, dtype="int32")), E_SHAPE, "positions"),
    (dict(q_weight=_zeros(63)), E_SHAPE, "q_weight"),
    (dict(k_weight=_zeros(3, 64)), E_SHAPE, "k_weight"),
    (dict(q=_zeros(6, 4, 68)[..., 2:66]), E_ALIGN, "16-byte"),
    (dict(k=_zeros(6, 2, 68)[..., :64]), E_ALIGN, "multiples of 16"),
    (dict(q_out=_zeros(6, 1, 64).expand(6, 4, 64)), E_ALIGN, "expanded"),
    (dict(k_pages=_zeros(1, 16, 2, 64).expand(7, 16, 2, 64)), E_ALIGN, "expanded"),
])
def test_paged_append_refuses(pkg, over, code, word):
    _refused(pkg, "l3d_paged_append", _append_args(**over), code, word)


def _paged_args(**over):
    B, N, Hq, Hkv, D = 3, 2, 4, 2, 64
    a = dict(q=_zeros(B, N, Hq, D), k_pages=_zeros(7, 16, Hkv, D), v_pages=_zeros(7, 16, Hkv, D),
             table=_zeros(B, 5, dtype="int32"), lengths=_zeros(B, dtype="int32"), scale=0.125,
             out=_zeros(B, N, Hq, D), workspace=256, bytes=1 << 30)
    assert not set(over) - set(a)
    return [*(a | over).values(), None]


@pytest.mark.parametrize("over,code,word", [
    (dict(q=None), E_NULL, "required"),
    (dict(lengths=None), E_NULL, "required"),
    (dict(q=_zeros(3, 2, 4, 64, dtype="float32")), E_DTYPE, "BF16"),
    (dict(v_pages=_zeros(7, 16, 2, 64, dtype="float16")), E_DTYPE, "F16"),
    (dict(q=_zeros(3, 4, 64)), E_SHAPE, "[B, N, H, D]"),
    (dict(q=_zeros(3, 2, 64, 4).transpose(2, 3)), E_ALIGN, "contiguous"),
    (dict(q=_zeros(3, 2, 4, 96), out=_zeros(3, 2, 4, 96)), E_UNSUPPORTED, "64 or 128"),
    (dict(out=_zeros(3, 1, 4, 64)), E_SHAPE, "out"),
    (dict(v_pages=_zeros(8, 16, 2, 64)), E_SHAPE, "k_pages and v_pages"),
    (dict(k_pages=_zeros(7, 16, 2, 128), v_pages=_zeros(7, 16, 2, 128)), E_SHAPE, "k_pages and v_pages"),
    (dict(q=_zeros(3, 2, 3, 64), out=_zeros(3, 2, 3, 64)), E_SHAPE, "multiple of the key heads"),
    (dict(table=_zeros(3, 5, dtype="int64")), E_DTYPE, "table"),
    (dict(table=_zeros(2, 5, dtype="int32")), E_SHAPE, "table"),
    (dict(table=_zeros(5, 3, dtype="int32").t()), E_SHAPE, "contiguous rows"),
    (dict(lengths=_zeros(3, dtype="float32")), E_DTYPE, "lengths"),
    (dict(lengths=_zeros(4, dtype="int32")), E_SHAPE, "lengths"),
    (dict(lengths=_zeros(6, dtype="int32")[::2]), E_SHAPE, "lengths"),
    (dict(scale=0.0), E_UNSUPPORTED, "scale"),
    (dict(scale=math.nan), E_UNSUPPORTED, "scale"),
    (dict(scale=2.9e38), E_UNSUPPORTED, "scale"),
    (dict(k_pages=_zeros(7, 0, 2, 64), v_pages=_zeros(7, 0, 2, 64)), E_UNSUPPORTED, "no tokens"),
    (dict(q=_zeros(4097, 1, 4, 64), out=_zeros(4097, 1, 4, 64), table=_zeros(4097, 5, dtype="int32"),
          lengths=_zeros(4097, dtype="int32")), E_UNSUPPORTED, "4096"),
    (dict(table=_zeros(3, 900, dtype="int32"), bytes=0), E_WORKSPACE, "workspace"),
    (dict(table=_zeros(3, 900, dtype="int32"), workspace=None), E_WORKSPACE, "workspace"),
    (dict(workspace=264), E_ALIGN, "256"),
    (dict(k_pages=_zeros(7, 16, 2, 68)[..., :64]), E_ALIGN, "multiples of 16"),
    (dict(k_pages=_zeros(1, 16, 2, 64).expand(7, 16, 2, 64)), E_ALIGN, "expanded"),
    (dict(out=_zeros(3, 2, 1, 64).expand(3, 2, 4, 64)), E_ALIGN, "out must not be expanded"),
    (dict(out=_zeros(1, 2, 4, 64).expand(3, 2, 4, 64)), E_ALIGN, "out must not be expanded"),
])
def test_paged_attention_refuses(pkg, over, code, word):
    _refused(pkg, "l3d_paged_attention", _paged_args(**over), code, word)


def test_nothing_to_do(pkg):
    """Empty batches are no error, and need no device."""
    L = pkg._lib
    e = {n: _zeros(0, 2, 4, 64) for n in ("q", "out")}
    args = _paged_args(**e, table=_zeros(0, 5, dtype="int32"), lengths=_zeros(0, dtype="int32"), workspace=None, bytes=0)
    assert L.lib().l3d_paged_attention(*[L.packed(a) if hasattr(a, "dim") else a for a in args]) == 0
    assert L.lib().l3d_paged_attention_workspace_size(0, 4, 2, 1, 80, 64) == 0
    assert L.lib().l3d_paged_attention_workspace_size(3, 5, 2, 1, 80, 64) == 0
    args = _append_args(q=_zeros(0, 4, 64), k=_zeros(0, 2, 64), v=_zeros(0, 2, 64), q_out=_zeros(0, 4, 64),
                        positions=_zeros(0, 2, dtype="int32"))
    assert L.lib().l3d_paged_append(*[L.packed(a) if hasattr(a, "dim") else a for a in args]) == 0


def test_rotary_axes(pkg):
    R = pkg.ops.RotaryAxes
    r = R(128, (16, 24, 24), theta=1e6, device="cpu")
    assert r.half == 64 and r.axes == 3 and r.axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    want = np.concatenate([1e6 ** (-np.arange(n) / n) for n in (16, 24, 24)])
    got = r.freqs.double().sum(1).numpy()
    assert np.abs(got / want - 1).max() < 2.0 ** -46  # the low part holds what the high one rounds off
    assert R(64, (16, 16), layout="axis", device="cpu").half == 16
    assert R(64, (5, 6), layout="interleaved", device="cpu").half == 0
    f = np.linspace(0.1, 1, 8)
    assert np.allclose(R(64, (8,), frequencies=f, device="cpu").freqs.double().sum(1).numpy(), f, rtol=1e-14)
    for bad, word in (((64, (33,)), "do not fit"), ((64, ()), "do not fit"), ((64, (0, 8)), "do not fit"),
                      ((64, (12,)), "multiple of 8"), ((64, (16, 8), 1e4, "axis"), "equal sections"),
                      ((64, (8,), 1e4, "pairs"), "unknown layout"), ((64, (8,), 1e4, "half", f[:7]), "8 finite"),
                      ((64, (8,), 1e4, "half", f * np.inf), "8 finite")):
        with pytest.raises(ValueError, match=word):
            R(*bad, device="cpu")


def test_front_end_refuses(pkg):
    ops = pkg.ops
    q, kv, pages = _zeros(2, 4, 64), _zeros(2, 2, 64), _zeros(3, 16, 2, 64)
    table, held = _zeros(2, 1, dtype="int32"), _zeros(2, dtype="int32")
    rope = ops.RotaryAxes(64, (16, 16), device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_append(q, kv, kv, pages, pages, table, held)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, pages, pages, table, held)
    with pytest.raises(ValueError, match="axes"):
        ops.paged_append(q, kv, kv, pages, pages, table, held, rope=rope, positions=_zeros(2, 3, dtype="int32"))
    with pytest.raises(ValueError, match="heads of 64"):
        ops.paged_append(q, kv, kv, pages, pages, table, held, rope=ops.RotaryAxes(128, (16,), device="cpu"))


def _cross_args(**over):
    Tq, Tk, Hq, Hkv, D = 60, 40, 4, 2, 64
    a = dict(q=_zeros(Tq, Hq, D), k=_zeros(Tk, Hkv, D), v=_zeros(Tk, Hkv, D), k_offsets=_zeros(4, dtype="int32"),
             q_offsets=_zeros(4, dtype="int64"), scale=0.125, out=_zeros(Tq, Hq, D), workspace=256, bytes=1 << 30)
    assert not set(over) - set(a)
    return [*(a | over).values(), None]


@pytest.mark.parametrize("over,code,word", [
    (dict(q=None), E_NULL, "required"),
    (dict(k_offsets=None), E_NULL, "required"),
    (dict(q=_zeros(60, 4, 64, dtype="float32")), E_DTYPE, "BF16"),
    (dict(v=_zeros(40, 2, 64, dtype="float16")), E_DTYPE, "F16"),
    (dict(q=_zeros(1, 60, 4, 64)), E_SHAPE, "[Tq, Hq, D]"),
    (dict(k=_zeros(40, 64, 2).transpose(1, 2)), E_ALIGN, "contiguous"),
    (dict(q=_zeros(60, 4, 80), out=_zeros(60, 4, 80)), E_UNSUPPORTED, "64 or 128"),
    (dict(out=_zeros(59, 4, 64)), E_SHAPE, "out"),
    (dict(v=_zeros(41, 2, 64)), E_SHAPE, "k and v"),
    (dict(k=_zeros(40, 2, 128), v=_zeros(40, 2, 128)), E_SHAPE, "k and v"),
    (dict(k=_zeros(40, 3, 64), v=_zeros(40, 3, 64)), E_SHAPE, "multiple of the key heads"),
    (dict(k_offsets=_zeros(4, dtype="float32")), E_SHAPE, "k_offsets"),
    (dict(k_offsets=_zeros(0, dtype="int32")), E_SHAPE, "k_offsets"),
    (dict(k_offsets=_zeros(8, dtype="int32")[::2]), E_SHAPE, "k_offsets"),
    (dict(q_offsets=_zeros(5, dtype="int32")), E_SHAPE, "q_offsets"),
    (dict(q_offsets=None, k_offsets=_zeros(8, dtype="int32")), E_SHAPE, "divide evenly"),
    (dict(q_offsets=None, k_offsets=_zeros(1, dtype="int32")), E_SHAPE, "divide evenly"),
    (dict(q_offsets=None, k_offsets=_zeros((1 << 20) + 2, dtype="int32"), q=_zeros(0, 4, 64), out=_zeros(0, 4, 64)),
     E_UNSUPPORTED, "2^20 sequences"),
    (dict(k_offsets=_zeros((1 << 20) + 1, dtype="int32"), q_offsets=_zeros((1 << 20) + 1, dtype="int32"),
          q=_zeros(1, 65, 64), out=_zeros(1, 65, 64), k=_zeros(1, 65, 64), v=_zeros(1, 65, 64)), E_UNSUPPORTED, "2^26"),
    (dict(scale=-1.0), E_UNSUPPORTED, "scale"),
    (dict(scale=math.nan), E_UNSUPPORTED, "scale"),
    (dict(scale=3e38), E_UNSUPPORTED, "scale"),
    (dict(q=_zeros(60, 258, 64), out=_zeros(60, 258, 64)), E_UNSUPPORTED, "128 query heads"),
    (dict(k=_zeros(1, 2, 64).expand(40, 2, 64)), E_ALIGN, "expanded"),
    (dict(q=_zeros(60, 1, 64).expand(60, 4, 64)), E_ALIGN, "expanded"),
    (dict(out=_zeros(60, 1, 64).expand(60, 4, 64)), E_ALIGN, "out must not be expanded"),
    (dict(out=_zeros(1, 4, 64).expand(60, 4, 64)), E_ALIGN, "out must not be expanded"),
    (dict(k=_zeros(4096, 2, 64), v=_zeros(4096, 2, 64), bytes=0), E_WORKSPACE, "workspace"),
    (dict(k=_zeros(4096, 2, 64), v=_zeros(4096, 2, 64), workspace=264), E_ALIGN, "256"),
    (dict(q_offsets=None, q=_zeros(3, 4, 64), out=_zeros(3, 4, 64), k=_zeros(9000, 2, 64), v=_zeros(9000, 2, 64),
          workspace=None), E_WORKSPACE, "workspace"),
    (dict(k=_zeros(40, 2, 68)[..., :64]), E_ALIGN, "multiples of 16"),
    (dict(q=_zeros(60, 4, 68)[..., 2:66]), E_ALIGN, "16-byte"),
])
def test_cross_attention_refuses(pkg, over, code, word):
    _refused(pkg, "l3d_cross_attention", _cross_args(**over), code, word)


def test_cross_attention_nothing_to_do(pkg):
    L = pkg._lib
    args = _cross_args(q=_zeros(0, 4, 64), out=_zeros(0, 4, 64), workspace=None, bytes=0)
    assert L.lib().l3d_cross_attention(*[L.packed(a) if hasattr(a, "dim") else a for a in args]) == 0
    size = L.lib().l3d_cross_attention_workspace_size
    assert size(0, 60, 40, 4, 2, 64, 1) == 0 and size(3, 60, 40, 4, 3, 64, 1) == 0 and size(3, 60, 0, 4, 2, 64, 1) == 0
    with pytest.raises(ValueError, match="CUDA"):
        pkg.ops.cross_attention(_zeros(3, 4, 64), _zeros(5, 4, 64), _zeros(5, 4, 64), _zeros(2, dtype="int32"))


@pytest.mark.parametrize("op", ["paged_attention", "cross_attention"])
def test_status_reaches_the_caller(pkg, monkeypatch, op):
    """A wait that ran out raises where it is asked for, as in the other serving entries."""
    from contextlib import nullcontext
    from types import SimpleNamespace

    import torch

    ops, seen = pkg.ops, []

    def call(name, *args):
        seen.append(name)
        args[0]._obj.value = 5

    monkeypatch.setattr(ops, "call", call)
    monkeypatch.setattr(ops, "invoke", lambda name, *a: seen.append(name))
    monkeypatch.setattr(torch.cuda, "device", lambda d: nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda d: SimpleNamespace(synchronize=lambda: seen.append("synchronised")))
    args = (_zeros(60, 4, 64), *[_zeros(40, 2, 64)] * 2, *[_zeros(4, dtype="int32")] * 2)
    getattr(ops, op)(*args)
    assert seen == [f"l3d_{op}"]
    with pytest.raises(pkg._lib.L3dError, match=f"l3d_{op}.*status word 5"):
        getattr(ops, op)(*args, check=True)
    assert seen[1:] == [f"l3d_{op}", "synchronised", "l3d_kernel_status"]


def test_native_calls_check_their_arguments(pkg):
    L = pkg._lib
    with pytest.raises(TypeError, match="tensor expected"):
        L.invoke("l3d_paged_append", 0, 1e-6, 0, *[None] * 14)
    with pytest.raises(ValueError, match="CUDA"):
        L.invoke("l3d_paged_append", 0, 1e-6, 0, *[None] * 11, _zeros(3), None, None)
    with pytest.raises(TypeError, match="tensor expected"):
        L.invoke("l3d_paged_append", 0, 1e-6, 0, 7, *[None] * 13)
    for name in ("l3d_paged_attention", "l3d_cross_attention"):
        with pytest.raises(TypeError, match="tensor expected"):
            L.invoke(name, L.address(name + "_workspace_size"), 0, 0.125, *[None] * 6)
        with pytest.raises(TypeError, match="10 arguments"):
            L.invoke(name, 0)
    with pytest.raises(TypeError, match="18 arguments"):
        L.invoke("l3d_paged_append", 0)
    with pytest.raises(TypeError):
        L.invoke("l3d_paged_append", 0, "eps", 0, *[None] * 14)


def test_calls_without_the_native_module_say_why(pkg):
    from test_serving_checks import _without_pack

    out = _without_pack("import torch\n"
                        "z, i = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)\n"
                        "for f in (lambda: pkg.ops.cross_attention(z, z, z, i), lambda: pkg.ops.paged_attention(z, z, z, i, i),\n"
                        "          lambda: pkg.ops.paged_append(z, z, z, z, z, i, i)):\n"
                        "    try: f()\n"
                        "    except RuntimeError as e: print(e)\n")
    assert out.count("made for another torch") == 3
