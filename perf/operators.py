"""Cases of the operators that serve a transformer block to many requests around one shared context.

Three operators: a projection with low-rank adapters of many requests (`lora`), attention over a prefix that
the whole batch shares plus each request's own keys (`prefix`), and the block seam with a norm on either
side of the residual (`seam`).  `run` computes each in plain torch operations in 32 bits, or, where `own`
is set, through this package's entry points; `exact` restates the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# Bounds of a drawn case's work: those of the largest listed cases.
MAX_LORA_FLOPS = 2 * 31569 * 8192 * 1536
MAX_SCORES = 4 * 12 * 4097 * (1029 + 4097)
MAX_KV = 160 << 20
MAX_SEAM = 131072 * 2048


def _lora(name, M, K, N, A, rank, per, act="none", residual=False):
    return {"name": name, "op": "lora", "M": M, "K": K, "N": N, "A": A, "rank": rank, "per": per, "act": act,
            "residual": residual}


def _prefix(name, B, Hq, Hkv, N, D, P, S, causal=False, dtype="bf16"):
    return {"name": name, "op": "prefix", "B": B, "Hq": Hq, "Hkv": Hkv, "N": N, "D": D, "P": P, "S": S,
            "causal": causal, "dtype": dtype}


def _seam(name, B, T, C, norm, ada, dtype="bf16"):
    return {"name": name, "op": "seam", "B": B, "T": T, "C": C, "norm": norm, "ada": ada, "dtype": dtype}


def listed():
    return [
        # One row for each of 16 requests (the timestep or modulation vectors of a serving batch): latency.
        _lora("adapters, 16 single rows", 16, 2048, 2048, 8, 16, "row"),
        # 64 rows whose adapters are mostly different, MLP up projection with its activation.
        _lora("adapters, 64 mixed rows", 64, 2048, 8192, 32, 64, "row", act="gelu_erf"),
        # The output projection of a batch of two requests of 2049 tokens, gated and added to the residual.
        _lora("adapters, two requests", 4098, 2048, 2048, 4, 32, "request", residual=True),
        # The MLP up projection over the voxel rows of a few scenes.
        _lora("adapters, voxel rows", 31569, 1536, 8192, 6, 64, "scene", act="gelu"),
        # A few new tokens per request behind an image's tokens, each seeing those before it.
        _prefix("prefix, few tokens causal", 4, 8, 2, 5, 64, 1029, 77, causal=True, dtype="f16"),
        # One new token for each of 64 requests behind a long common context, own keys of ragged lengths.
        _prefix("prefix, one token long", 64, 16, 4, 1, 128, 32768, 512),
        # Eight variants generated from one image: cross attention to the image's tokens.
        _prefix("prefix, variants of an image", 8, 16, 16, 2049, 128, 1370, 0),
        # Joint attention of four scenes' own tokens and a shared condition.
        _prefix("prefix, joint tokens", 4, 12, 12, 4097, 128, 1029, 4097, dtype="f16"),
        # The seam of a batch of single rows: latency.
        _seam("seam, 8 single rows", 8, 1, 2048, "rms", True),
        # The seam of a scene of eight views with affine LayerNorms and a LayerScale.
        _seam("seam, eight views", 8, 1374, 1024, "layer", False),
        # The seam of a batch of two requests in 32 bits.
        _seam("seam, two requests in 32 bits", 2, 2049, 2048, "layer", True, dtype="f32"),
        # The seam of a large batch.
        _seam("seam, large batch", 64, 2048, 2048, "rms", True),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm; 3072, a size that no configuration here has, is
    drawn again."""
    got = max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) // step * step)
    return got if got != 3072 else _log(rng, lo, hi, step)


def _drawn(c):
    del c["name"]
    return c


def draw(rng):
    op = rng.choice(["lora", "prefix", "seam"])
    if op == "lora":
        M, K, N = _log(rng, 1, 31569), _log(rng, 256, 4096, 8), _log(rng, 64, 8192, rng.choice([1, 64]))
        M = max(1, min(M, MAX_LORA_FLOPS // (2 * K * N)))
        A, rank = _log(rng, 1, 32), rng.choice([4, 8, 16, 24, 32, 64])
        per = rng.choice(["row", "request", "scene"]) if M < 1024 else rng.choice(["request", "scene"])
        return _drawn(_lora("", M, K, N, A, rank, per, rng.choice(["none", "gelu", "gelu_erf", "silu"]),
                            rng.random() < 0.4))
    if op == "prefix":
        D, Hkv, G = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4, 8])
        B, N = _log(rng, 1, 64), rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 4097)])
        P, S = _log(rng, 1, 32768), rng.choice([0, _log(rng, 1, 512), _log(rng, 1, 4097)])
        P = max(1, min(P, MAX_KV // (4 * Hkv * D)))
        S = min(S, MAX_KV // (4 * Hkv * D * B))
        N = max(1, min(N, MAX_SCORES // (B * Hkv * G * (P + S))))
        return _drawn(_prefix("", B, Hkv * G, Hkv, N, D, P, S, S >= N and rng.random() < 0.4,
                              rng.choice(["bf16", "f16"])))
    C = _log(rng, 64, 8192, rng.choice([1, 64, 64]))
    rows = min(_log(rng, 1, 131072), MAX_SEAM // C)
    B = min(rows, _log(rng, 1, 64))
    return _drawn(_seam("", B, rows // B, C, rng.choice(["rms", "layer"]), rng.random() < 0.5,
                        rng.choice(["bf16", "bf16", "f16", "f32"])))


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _ranks(c):
    """Ranks of the adapters: the largest one, and others below it."""
    r = random.Random(c["A"] * 1000 + c["rank"])
    return [c["rank"] if i == 0 else r.choice([c["rank"], max(1, c["rank"] // 2), max(1, c["rank"] // 4)])
            for i in range(c["A"])]


def _requests(M):
    """Equal requests that M rows divide into."""
    return next(n for n in (2, 3, 5, 7, 1) if M % n == 0)


def _lengths(c):
    """Own keys that each request holds: ragged, the longest fills the cache."""
    r = random.Random(c["B"] * 7919 + c["S"])
    got = [r.randint(min(c["S"], c["N"]) if c["causal"] else 0, c["S"]) for _ in range(c["B"])]
    got[0] = c["S"]
    return got


def _lora_inputs(c, seed):
    g = _gen(seed)
    M, K, N, A = c["M"], c["K"], c["N"], c["A"]
    s = {"x": _randn(g, (M, K), torch.bfloat16), "w": _randn(g, (N, K), torch.bfloat16, K ** -0.5),
         "bias": _randn(g, (N,), std=0.1), "ranks": _ranks(c)}
    R = max(s["ranks"])
    s["a"] = _randn(g, (A, R, K), torch.bfloat16, K ** -0.5)
    s["b"] = _randn(g, (A, N, R), torch.bfloat16, 0.5 * R ** -0.5)
    for i, r in enumerate(s["ranks"]):
        s["a"][i, r:] = 0
        s["b"][i, :, r:] = 0
    s["scales"] = [0.5 + 0.25 * (i % 5) for i in range(A)]
    s["scale"] = torch.tensor(s["scales"], device="cuda")
    if c["per"] == "row":  # any adapter, or none, for each row
        ids = torch.randint(-1, A, (M,), generator=g, device="cuda")
    elif c["per"] == "request":  # rows in equal requests
        ids = torch.randint(-1, A, (_requests(M),), generator=g, device="cuda")
    else:  # consecutive stretches of rows of uneven lengths
        cuts = torch.randint(0, M + 1, (A,), generator=g, device="cuda")
        row = torch.arange(M, device="cuda")
        ids = (row[:, None] >= cuts[None, :]).sum(1) - 1
    s["ids"] = ids.to(torch.int32)
    if c["residual"]:
        s["residual"] = _randn(g, (M, N), torch.bfloat16)
        s["gate"] = _randn(g, (N,), std=0.3, mean=0.5)
    return s


def _prefix_inputs(c, seed):
    g = _gen(seed)
    dt, B, D, H = DTYPES[c["dtype"]], c["B"], c["D"], c["Hkv"]
    # Token-major memory seen as [B, H, N, D], as projections leave it.
    s = {"q": _randn(g, (B, c["N"], c["Hq"], D), dt).transpose(1, 2),
         "pk": _randn(g, (c["P"], H, D), dt).transpose(0, 1), "pv": _randn(g, (c["P"], H, D), dt).transpose(0, 1)}
    if c["S"]:
        s["k"] = _randn(g, (B, H, c["S"], D), dt)
        s["v"] = _randn(g, (B, H, c["S"], D), dt)
        s["lengths"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)
    return s


def _seam_inputs(c, seed):
    g = _gen(seed)
    dt, B, T, C = DTYPES[c["dtype"]], c["B"], c["T"], c["C"]
    s = {"x": _randn(g, (B, T, C), dt), "h": _randn(g, (B, T, C), dt, 2.0, 0.1),
         "post_weight": _randn(g, (C,), dt, 0.1, 1.0), "weight": _randn(g, (C,), dt, 0.1, 1.0),
         "res_scale": 0.875}
    if c["norm"] == "layer":
        s["post_bias"], s["bias"] = _randn(g, (C,), dt, 0.1), _randn(g, (C,), dt, 0.1)
    if c["ada"]:  # chunks of one vector per request
        vec = _randn(g, (B, 3 * C), dt, 0.2)
        s["gate"], s["shift"], s["scale"] = vec.chunk(3, -1)
    else:
        s["gate"] = _randn(g, (C,), dt, 0.1, 0.5)
    return s


_INPUTS = {"lora": _lora_inputs, "prefix": _prefix_inputs, "seam": _seam_inputs}


def prepare(case, seed):
    s = _INPUTS[case["op"]](case, seed)
    s["case"] = case
    if own:
        import __graft_entry__

        s["ops"] = __graft_entry__.load_package().ops
        if case["op"] == "lora":  # the served adapters, laid out once as a server keeps them
            s["adapters"] = s["ops"].LoraAdapters([a[:r] for a, r in zip(s["a"], s["ranks"])],
                                                  [b[:, :r] for b, r in zip(s["b"], s["ranks"])], s["scales"])
    return s


# -------------------------------------------------------------- plain forms
def _act(name, z):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    if name == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    return z


def _plain_lora(c, s):
    M, A = c["M"], c["A"]
    x = s["x"].float()
    ids = s["ids"].repeat_interleave(M // s["ids"].numel())
    mine = ids[:, None] == torch.arange(A, device=ids.device, dtype=ids.dtype)
    t = (x @ s["a"].float().flatten(0, 1).T).view(M, A, -1) * (mine * s["scale"])[:, :, None]
    z = x @ s["w"].float().T + s["bias"] + t.flatten(1) @ s["b"].float().transpose(1, 2).flatten(0, 1)
    y = _act(c["act"], z)
    if c["residual"]:
        y = s["residual"].float() + s["gate"] * y
    return y.to(torch.bfloat16)


def _plain_prefix(c, s):
    B, H, G, N, D, P, S = c["B"], c["Hkv"], c["Hq"] // c["Hkv"], c["N"], c["D"], c["P"], c["S"]
    q = s["q"].float().reshape(B, H, G * N, D) * D ** -0.5
    score = q @ s["pk"].float().transpose(-1, -2)
    if S:
        row, key = torch.arange(N, device=q.device), torch.arange(S, device=q.device)
        last = s["lengths"][:, None] - N + row if c["causal"] else (s["lengths"] - 1)[:, None].expand(B, N)
        seen = (key <= last[:, :, None])[:, None, None].expand(B, 1, G, N, S).reshape(B, 1, G * N, S)
        mine = q @ s["k"].float().transpose(-1, -2)
        score = torch.cat([score, torch.where(seen, mine, -math.inf)], -1)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = p[..., :P] @ s["pv"].float()
    if S:
        o = o + p[..., P:] @ s["v"].float()
    return (o / total).to(s["q"].dtype).view(B, H * G, N, D)


def _plain_norm(kind, v, w, b):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w.float()
    return v if b is None else v + b.float()


def _plain_seam(c, s):
    n = _plain_norm(c["norm"], s["h"].float(), s["post_weight"], s.get("post_bias"))
    gate = s["gate"].float()
    r = s["res_scale"] * s["x"].float() + (gate[:, None] if c["ada"] else gate) * n
    y = _plain_norm(c["norm"], r, s["weight"], s.get("bias"))
    if c["ada"]:
        y = y * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
    return {"r": r.to(s["x"].dtype), "y": y.to(s["x"].dtype)}


_PLAIN = {"lora": _plain_lora, "prefix": _plain_prefix, "seam": _plain_seam}


def _own(c, s):
    ops = s["ops"]
    if c["op"] == "lora":
        return ops.lora_linear(s["x"], s["w"], s["adapters"], s["ids"], bias=s["bias"],
                               act=None if c["act"] == "none" else c["act"], residual=s.get("residual"),
                               gate=s.get("gate"))
    if c["op"] == "prefix":
        return ops.shared_prefix_attention(s["q"], s["pk"], s["pv"], s.get("k"), s.get("v"), s.get("lengths"),
                                           causal=c["causal"])
    r, y = ops.sandwich_residual_norm(s["x"], s["h"], post_weight=s["post_weight"], post_bias=s.get("post_bias"),
                                      gate=s["gate"], res_scale=s["res_scale"], weight=s["weight"],
                                      bias=s.get("bias"), shift=s.get("shift"), scale=s.get("scale"),
                                      norm=c["norm"], eps=1e-6)
    return {"r": r, "y": y}


def run(state):
    c = state["case"]
    return _own(c, state) if own else _PLAIN[c["op"]](c, state)


# ------------------------------------------------------------------- 64 bits
def _exact_lora(c, s):
    x = s["x"].double()
    z = torch.addmm(s["bias"].double(), x, s["w"].double().T)
    per = c["M"] // s["ids"].numel()
    at = s["ids"].long()[torch.arange(c["M"], device=x.device) // per]
    for i, r in enumerate(s["ranks"]):
        rows = torch.nonzero(at == i)[:, 0]
        down = x[rows] @ s["a"][i, :r].double().T
        z[rows] += s["scales"][i] * (down @ s["b"][i, :, :r].double().T)
    if c["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif c["act"] == "gelu":
        z = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    elif c["act"] == "gelu_erf":
        z = 0.5 * z * torch.erfc(-z / math.sqrt(2))
    return s["residual"].double() + s["gate"].double() * z if c["residual"] else z


def _exact_prefix(c, s):
    G, N = c["Hq"] // c["Hkv"], c["N"]
    out = torch.empty(c["B"], c["Hq"], N, c["D"], dtype=torch.float64, device="cuda")
    lens = _lengths(c) if c["S"] else [0] * c["B"]
    for b in range(c["B"]):
        for h in range(c["Hkv"]):
            k, v = s["pk"][h].double(), s["pv"][h].double()
            if c["S"]:
                k = torch.cat([k, s["k"][b, h, :lens[b]].double()])
                v = torch.cat([v, s["v"][b, h, :lens[b]].double()])
            q = s["q"][b, h * G:(h + 1) * G].double()
            w = torch.einsum("gnd,sd->gns", q, k) / math.sqrt(c["D"])
            if c["causal"]:  # row i sees the own keys up to its own place
                future = torch.arange(k.shape[0], device=k.device) - c["P"] > \
                    torch.arange(N, device=k.device)[:, None] + lens[b] - N
                w = w.masked_fill(future, -math.inf)
            out[b, h * G:(h + 1) * G] = torch.softmax(w, -1) @ v
    return out


def _exact_seam(c, s):
    def norm(v, w, b):
        mean = v.mean(-1, keepdim=True) if c["norm"] == "layer" else 0.0
        std = torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + 1e-6)
        return (v - mean) / std * w.double() + (0.0 if b is None else b.double())

    def vec(t):
        return t.double().reshape(-1, 1, c["C"])

    r = s["res_scale"] * s["x"].double() + vec(s["gate"]) * norm(s["h"].double(), s["post_weight"], s.get("post_bias"))
    y = norm(r, s["weight"], s.get("bias"))
    if c["ada"]:
        y = y * (1 + vec(s["scale"])) + vec(s["shift"])
    return {"r": r, "y": y}


_EXACT = {"lora": _exact_lora, "prefix": _exact_prefix, "seam": _exact_seam}


def exact(case, seed):
    return _EXACT[case["op"]](case, _INPUTS[case["op"]](case, seed))


# ---------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "lora":
        M, K, N, ranks = c["M"], c["K"], c["N"], _ranks(c)
        used = min(c["A"], M) if c["per"] != "request" else min(c["A"], _requests(M))
        low = sum(sorted(ranks)[:used])  # rows of A and columns of B that the rows in use read
        out = 2 * M * N
        return {"bytes": 2 * M * K + 2 * N * K + 2 * low * (N + K) + 4 * N + out * (2 if c["residual"] else 1),
                "flops": 2 * M * N * K + 2 * M * (sum(ranks) / len(ranks)) * (N + K)}
    if c["op"] == "prefix":
        lens = _lengths(c) if c["S"] else [0] * c["B"]
        own_pairs = sum(sum(min(n, max(0, n - c["N"] + i + 1)) for i in range(c["N"])) if c["causal"] else n * c["N"]
                        for n in lens)
        pairs = c["Hq"] * (c["B"] * c["N"] * c["P"] + own_pairs)
        kv = c["Hkv"] * c["D"] * 2 * (c["P"] + sum(lens))
        return {"bytes": 2 * (2 * c["B"] * c["Hq"] * c["N"] * c["D"] + kv), "flops": 4 * c["D"] * pairs}
    n = c["B"] * c["T"] * c["C"]
    vectors = c["C"] * ((4 if c["norm"] == "layer" else 2) + (3 * c["B"] if c["ada"] else 1))
    return {"bytes": SIZE[c["dtype"]] * (4 * n + vectors), "flops": 20 * n}
