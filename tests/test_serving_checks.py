"""CPU: the entries that serve many requests (adapters, shared prefixes,
sandwich norms) refuse invalid requests on the host, before any launch."""
import math

import pytest

E_SHAPE, E_DTYPE, E_ALIGN, E_UNSUPPORTED, E_NULL, E_WORKSPACE = 1, 2, 3, 4, 6, 7


def _zeros(*shape, dtype="bfloat16"):
    import torch

    return torch.zeros(shape, dtype=getattr(torch, dtype))


def _refused(pkg, name, args, code, word):
    lib = pkg._lib.lib()
    args = [pkg._lib.packed(a) if a is None or hasattr(a, "dim") else a for a in args]
    assert getattr(lib, name)(*args) == code, lib.l3d_last_error()
    assert word in lib.l3d_last_error().decode()


def _lora_args(**over):
    m, n, k, r = 12, 40, 64, 16
    a = dict(x=_zeros(m, k), weight=_zeros(n, k), bias=None, lora_a=_zeros(3, r, k),
             lora_b=_zeros(3, n, r), lora_scale=_zeros(3, dtype="float32"), ranks=None,
             ids=_zeros(m, dtype="int32"), act=0, residual=None, gate=None, y=_zeros(m, n),
             workspace=256, bytes=1 << 20)
    assert not set(over) - set(a)
    return [*(a | over).values(), None]


@pytest.mark.parametrize("over,code,word", [
    (dict(x=None), E_NULL, "x is required"),
    (dict(ids=None), E_NULL, "ids is required"),
    (dict(x=_zeros(12, 64, dtype="float16")), E_DTYPE, "BF16"),
    (dict(y=_zeros(12, 40, dtype="float16")), E_DTYPE, "y must be"),
    (dict(lora_scale=_zeros(3)), E_DTYPE, "lora_scale"),
    (dict(ids=_zeros(12, dtype="float32")), E_DTYPE, "ids"),
    (dict(ids=_zeros(5, dtype="int32")), E_SHAPE, "divide evenly"),
    (dict(ids=_zeros(0, dtype="int32")), E_SHAPE, "ids"),
    (dict(lora_a=_zeros(3, 8, 64), lora_b=_zeros(3, 40, 8)), E_UNSUPPORTED, "multiple of 16"),
    (dict(lora_a=_zeros(3, 272, 64), lora_b=_zeros(3, 40, 272)), E_UNSUPPORTED, "at most 256"),
    (dict(lora_b=_zeros(3, 16, 40)), E_SHAPE, "lora_b"),
    (dict(lora_b=_zeros(2, 40, 16)), E_SHAPE, "lora_b"),
    (dict(y=_zeros(12, 41)), E_SHAPE, "y last dim"),
    (dict(y=_zeros(11, 40)), E_SHAPE, "leading dims"),
    (dict(weight=_zeros(40, 60), x=_zeros(12, 60), lora_a=_zeros(3, 16, 60)), E_ALIGN, "multiple of 8"),
    (dict(x=_zeros(12, 68)[:, 2:66]), E_ALIGN, "16-byte"),
    (dict(ranks=_zeros(3, dtype="int64")), E_DTYPE, "ranks"),
    (dict(ranks=_zeros(4, dtype="int32")), E_SHAPE, "ranks"),
    (dict(act=9), E_UNSUPPORTED, "activation"),
    (dict(bias=_zeros(39)), E_SHAPE, "bias"),
    (dict(residual=_zeros(12, 40, dtype="float32")), E_DTYPE, "residual"),
    (dict(residual=_zeros(12, 39)), E_SHAPE, "residual"),
    (dict(gate=_zeros(40)), E_SHAPE, "needs a residual"),
    (dict(bytes=0), E_WORKSPACE, "workspace"),
    (dict(workspace=None), E_WORKSPACE, "workspace"),
    (dict(workspace=264), E_ALIGN, "256"),
])
def test_lora_linear_refuses(pkg, over, code, word):
    _refused(pkg, "l3d_lora_linear", _lora_args(**over), code, word)


def _prefix_args(**over):
    B, H, Hkv, N, P, S, D = 2, 4, 2, 3, 70, 9, 64
    a = dict(q=_zeros(B, H, N, D), prefix_k=_zeros(Hkv, P, D), prefix_v=_zeros(Hkv, P, D),
             k=_zeros(B, Hkv, S, D), v=_zeros(B, Hkv, S, D), lengths=_zeros(B, dtype="int32"), causal=0,
             scale=0.125, out=_zeros(B, H, N, D), workspace=256, bytes=1 << 30)
    assert not set(over) - set(a)
    return [*(a | over).values(), None]


@pytest.mark.parametrize("over,code,word", [
    (dict(q=None), E_NULL, "required"),
    (dict(v=None), E_NULL, "together"),
    (dict(k=None, v=None), E_SHAPE, "need own keys"),
    (dict(k=None, v=None, lengths=None, causal=1), E_SHAPE, "need own keys"),
    (dict(q=_zeros(2, 4, 3, 64, dtype="float32")), E_DTYPE, "BF16"),
    (dict(prefix_k=_zeros(2, 70, 64, dtype="float16")), E_DTYPE, "F16"),
    (dict(q=_zeros(4, 3, 64)), E_SHAPE, "[B, H, N, D]"),
    (dict(q=_zeros(2, 4, 64, 3).transpose(2, 3)), E_ALIGN, "head dim"),
    (dict(q=_zeros(2, 4, 3, 32)), E_UNSUPPORTED, "64 or 128"),
    (dict(out=_zeros(2, 4, 4, 64)), E_SHAPE, "out"),
    (dict(prefix_v=_zeros(2, 71, 64)), E_SHAPE, "prefix_k"),
    (dict(k=_zeros(2, 2, 8, 64)), E_SHAPE, "k and v"),
    (dict(q=_zeros(2, 3, 3, 64), out=_zeros(2, 3, 3, 64)), E_SHAPE, "multiple of the key heads"),
    (dict(lengths=_zeros(3, dtype="int32")), E_SHAPE, "lengths"),
    (dict(lengths=_zeros(2, dtype="float32")), E_DTYPE, "lengths"),
    (dict(scale=0.0), E_UNSUPPORTED, "scale"),
    (dict(scale=math.nan), E_UNSUPPORTED, "scale"),
    (dict(scale=math.inf), E_UNSUPPORTED, "scale"),
    (dict(prefix_k=_zeros(2, 4096, 64), prefix_v=_zeros(2, 4096, 64), bytes=0), E_WORKSPACE, "workspace"),
    (dict(prefix_k=_zeros(2, 4096, 64), prefix_v=_zeros(2, 4096, 64), workspace=264), E_ALIGN, "256"),
    (dict(k=_zeros(2, 2, 9, 68)[..., :64]), E_ALIGN, "multiples of 16"),
    (dict(k=_zeros(2, 2, 1, 64).expand(2, 2, 9, 64)), E_ALIGN, "expanded"),
])
def test_shared_prefix_attention_refuses(pkg, over, code, word):
    _refused(pkg, "l3d_shared_prefix_attention", _prefix_args(**over), code, word)


def _seam_args(**over):
    a = dict(x=_zeros(2, 5, 48), h=_zeros(2, 5, 48), norm=2, post_weight=None, post_bias=None, gate=None,
             res_scale=1.0, weight=None, bias=None, shift=None, scale=None, post_eps=1e-6, eps=1e-6,
             r_out=_zeros(2, 5, 48), y=_zeros(2, 5, 48))
    assert not set(over) - set(a)
    return [*(a | over).values(), None]


@pytest.mark.parametrize("over,code,word", [
    (dict(h=None), E_NULL, "required"),
    (dict(r_out=None), E_NULL, "required"),
    (dict(x=_zeros(2, 5, 48, dtype="int32")), E_DTYPE, "x must be"),
    (dict(h=_zeros(2, 5, 48, dtype="float16")), E_DTYPE, "h dtype"),
    (dict(y=_zeros(2, 5, 47)), E_SHAPE, "y shape"),
    (dict(h=_zeros(2, 48, 5).transpose(1, 2)), E_ALIGN, "h last dim"),
    (dict(norm=0), E_UNSUPPORTED, "norm"),
    (dict(y=None, weight=_zeros(48)), E_NULL, "need y"),
    (dict(eps=-1.0), E_UNSUPPORTED, "eps"),
    (dict(post_eps=math.nan), E_UNSUPPORTED, "eps"),
    (dict(post_weight=_zeros(47)), E_SHAPE, "post_weight"),
    (dict(gate=_zeros(3, 48)), E_SHAPE, "gate"),
    (dict(x=_zeros(1, 1, 24577), h=_zeros(1, 1, 24577), r_out=_zeros(1, 1, 24577), y=None),
     E_UNSUPPORTED, "row length"),
])
def test_sandwich_residual_norm_refuses(pkg, over, code, word):
    _refused(pkg, "l3d_sandwich_residual_norm", _seam_args(**over), code, word)


def test_front_end_refuses_host_tensors(pkg):
    ops = pkg.ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.LoraAdapters([_zeros(4, 64)], [_zeros(40, 4)])
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_prefix_attention(_zeros(1, 2, 3, 64), _zeros(2, 5, 64), _zeros(2, 5, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.sandwich_residual_norm(_zeros(2, 64), _zeros(2, 64))


def test_workspace_sizes_without_a_device(pkg):
    lib = pkg._lib.lib()
    assert lib.l3d_lora_linear_workspace_size(4098, 32) >= 4098 * 32 * 4
    assert lib.l3d_lora_linear_workspace_size(-1, 32) == 0
    # An empty batch has nothing to join.
    assert lib.l3d_shared_prefix_attention_workspace_size(0, 8, 2, 5, 1029, 77, 64) == 0


def test_descriptors_as_bytes(pkg):
    """The native descriptors are the ctypes ones; views keep their strides."""
    import torch

    L = pkg._lib
    for t in (_zeros(4, 5, 6).transpose(0, 2)[1:], _zeros(7, dtype="int64")[3:], _zeros(2, 0, 3), _zeros(1, 4).expand(3, 4),
              torch.zeros((), dtype=torch.uint8)):
        got, want = L.L3dTensor.from_buffer_copy(L.packed(t)), L.desc(t)
        assert (got.dtype, got.ndim) == (want.dtype, want.ndim)
        assert list(got.dims)[:t.dim()] == list(t.shape) and list(got.strides)[:t.dim()] == list(t.stride())
        assert (got.data or 0) + got.offset * t.element_size() == t.data_ptr()
    assert L.packed(None) is None
    with pytest.raises(TypeError):
        L.packed(3)
    with pytest.raises(TypeError, match="dtype"):
        L.packed(_zeros(2, dtype="float64"))
    with pytest.raises(ValueError, match="rank 7"):
        L.packed(_zeros(1, 1, 1, 1, 1, 1, 1))
    with pytest.raises(ValueError, match="CUDA"):
        L.packs(None, _zeros(2))


@pytest.mark.parametrize("name,shape", [("residual", (3, 2, 40)), ("residual", (6, 1, 40)), ("out", (3, 2, 40))])
def test_lora_linear_refuses_rows_in_another_order(pkg, name, shape):
    """As many rows under other leading dims than x's are other rows."""
    from types import SimpleNamespace

    ad = SimpleNamespace(rank=16, _desc=(None,) * 4)
    with pytest.raises(ValueError, match=f"{name} has leading dims"):
        pkg.ops.lora_linear(_zeros(2, 3, 64), _zeros(40, 64), ad, _zeros(2, dtype="int32"), **{name: _zeros(*shape)})


@pytest.mark.parametrize("scale", [2.4e38, 2.9e38, 3.3e38])
def test_shared_prefix_attention_refuses_a_scale_that_overflows(pkg, scale):
    """The kernel multiplies by scale * log2(e): finite scales whose product is not."""
    _refused(pkg, "l3d_shared_prefix_attention", _prefix_args(scale=scale), E_UNSUPPORTED, "scale")


@pytest.mark.parametrize("op", ["lora_linear", "shared_prefix_attention", "sandwich_residual_norm"])
def test_expired_waits_reach_the_caller(pkg, monkeypatch, op):
    """A status word of 5 raises where it is asked for, by argument or for all calls,
    and is read after the stream of the call has finished."""
    from contextlib import nullcontext
    from types import SimpleNamespace

    import torch

    ops, seen = pkg.ops, []

    def call(name, *args):
        seen.append(name)
        if name == "l3d_kernel_status":
            args[0]._obj.value = 5

    monkeypatch.setattr(ops, "call", call)
    monkeypatch.setattr(ops, "packs", lambda *a: a)
    monkeypatch.setattr(ops, "stream_of", lambda t: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda d: SimpleNamespace(synchronize=lambda: seen.append("synchronised")))
    args = {"lora_linear": (_zeros(2, 64), _zeros(40, 64), SimpleNamespace(rank=16, _desc=()), None),
            "shared_prefix_attention": (_zeros(1, 2, 3, 64), _zeros(2, 5, 64), _zeros(2, 5, 64)),
            "sandwich_residual_norm": (_zeros(2, 64), _zeros(2, 64))}[op]
    entry = f"l3d_{op}"
    getattr(ops, op)(*args)
    assert seen == [entry]  # a call does not wait unless it is asked to
    for by_argument in (True, False):
        seen.clear()
        monkeypatch.setattr(ops, "CHECK_STATUS", not by_argument)
        with pytest.raises(pkg._lib.L3dError, match=f"{entry}.*status word 5"):
            getattr(ops, op)(*args, **({"check": True} if by_argument else {}))
        assert seen == [entry, "synchronised", "l3d_kernel_status"]
    getattr(ops, op)(*args, check=False)
    assert seen[-1] == entry


def _without_pack(code):
    """Runs `code` in a process where _l3dpack cannot be imported."""
    import subprocess
    import sys
    from conftest import ROOT

    head = ("import sys\n"
            "class Refuse:\n"
            "    def find_spec(self, name, path=None, target=None):\n"
            "        if name.endswith('_l3dpack'): raise ImportError('undefined symbol: made for another torch')\n"
            "sys.meta_path.insert(0, Refuse())\n"
            "import __graft_entry__ as g\n"
            "pkg = g.load_package()\n")
    r = subprocess.run([sys.executable, "-c", head + code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_package_imports_without_the_native_descriptors(pkg):
    """Entries that do not use them, GGUF reading and the library's own checks are there."""
    out = _without_pack("import ctypes\n"
                        "L = pkg._lib\n"
                        "assert L.lib().l3d_abi_version() > 0\n"
                        "assert pkg.gguf and L.lib().l3d_layer_norm(None, None, None, 1e-5, None, None) == 6\n"
                        "print(L.lib().l3d_last_error().decode())\n")
    assert out.strip()


def test_calls_that_need_the_native_descriptors_say_why(pkg):
    out = _without_pack("import torch\n"
                        "z = torch.zeros(2, 5, 64, dtype=torch.bfloat16)\n"
                        "for f in (lambda: pkg.ops.sandwich_residual_norm(z, z), lambda: pkg._lib.packed(z),\n"
                        "          lambda: pkg.ops.shared_prefix_attention(z[None], z, z)):\n"
                        "    try: f()\n"
                        "    except RuntimeError as e: print(e)\n")
    assert out.count("made for another torch") == 3 and out.count("build.py") == 3


def test_native_descriptors_are_rebuilt_for_another_torch(pkg, monkeypatch, tmp_path):
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("l3d_build", Path(pkg.__file__).parent / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.BUILD, b.PACK = tmp_path, tmp_path / "_l3dpack.so"
    assert b._pack_needs()
    b.PACK.write_bytes(b"")
    assert b._pack_needs()  # of unknown origin
    (tmp_path / "_l3dpack.for").write_text(b._pack_for())
    assert not b._pack_needs()
    monkeypatch.setattr(b.importlib.metadata, "version", lambda name: "0.1")
    assert b._pack_needs()
