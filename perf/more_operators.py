"""Cases of the operators of a block that decodes tokens over a paged cache and an encoder's states.

Three operators: the new tokens' queries and keys normed per head, rotated by their positions and the keys and
values put into a paged cache (`append`), attention of a request's newest tokens over its pages (`paged`), and
attention of packed sequences to encoder states of other lengths (`cross`).  `run` computes each in plain torch
operations, or, where `own` is set, through this package's entry points; `exact` restates the definitions in
64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6

# Bounds of a drawn case's work: those of the largest listed cases.
MAX_TOKENS = 49152 * 24 * 128   # elements of q, k and v
MAX_KEYS = 8 * 65536 * 4 * 128  # elements of the keys read
MAX_PAIRS = 12 * 128 * 3 * 31569 * 1370
MAX_HELD = 64 * 4096 * 4 * 128  # elements of the keys held already


def _append(name, B, T, Hq, Hkv, D, page, sections, layout="half", norm=True, dtype="bf16", held=0):
    """T tokens of B requests (one each where T == B, else ragged) behind up to `held` tokens; positions on
    len(sections) axes, sections[a] pairs each."""
    return {"name": name, "op": "append", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "sections": "-".join(map(str, sections)), "layout": layout, "norm": norm, "dtype": dtype, "held": held}


def _paged(name, B, N, Hq, Hkv, D, page, S, dtype="bf16", ragged=True):
    return {"name": name, "op": "paged", "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "S": S,
            "ragged": ragged, "dtype": dtype}


def _cross(name, B, N, Hq, Hkv, D, S, rows="equal", dtype="bf16"):
    """B sequences of N rows each ("equal"), or of 1 .. N rows ("ragged"); encoder states of up to S rows each."""
    return {"name": name, "op": "cross", "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "S": S, "rows": rows,
            "dtype": dtype}


def listed():
    return [
        # One token of one request: latency.
        _append("append one token", 1, 1, 8, 2, 64, 16, (32,), held=300),
        # One token for each of 64 requests, placed in a video (time, height, width).
        _append("append 64 requests", 64, 64, 16, 4, 128, 16, (16, 24, 24), held=4096),
        # The views of five scenes arriving at once, positions on an image's axes, each axis a block of its own.
        _append("append views of scenes", 5, 10992, 16, 16, 64, 64, (16, 16), layout="axis", dtype="f16", held=1374),
        # Long prompts of 24 requests, pairs of neighbours rotated, part of the head left as it is, no norms.
        _append("append long prompts", 24, 49152, 16, 4, 128, 32, (48,), layout="interleaved", norm=False, held=100),
        # One token of one request with a short cache: latency.
        _paged("paged one request", 1, 1, 8, 2, 64, 16, 300),
        # One token for each of 64 requests, caches of ragged lengths.
        _paged("paged 64 requests", 64, 1, 16, 4, 128, 16, 4096),
        # A few tokens for each of 12 requests, a key head for each query head, pages of an odd size.
        _paged("paged few tokens", 12, 4, 12, 12, 128, 48, 4097, dtype="f16"),
        # One token for each of 8 requests behind very long caches.
        _paged("paged long caches", 8, 1, 16, 4, 128, 64, 65536, ragged=False),
        # A few short sequences beside encoders of about a sentence's length: latency.
        _cross("cross short sequences", 3, 70, 8, 2, 64, 77, rows="ragged", dtype="f16"),
        # One decoded token of each of 32 requests over its own image's tokens.
        _cross("cross single rows", 32, 1, 16, 16, 64, 1370),
        # Two objects of 2049 tokens, whose images gave different numbers of tokens.
        _cross("cross two objects", 2, 2049, 16, 16, 128, 1370),
        # The voxel rows of three scenes, each with an image of its own.
        _cross("cross voxel scenes", 3, 31569, 12, 12, 128, 1370),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) // step * step)


def _drawn(c):
    del c["name"]
    return c


def draw(rng):
    op = rng.choice(["append", "paged", "cross"])
    D, Hkv, G = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4, 8])
    dtype, page = rng.choice(["bf16", "bf16", "f16"]), rng.choice([1, 8, 16, 16, 32, 48, 64, 128, 256])
    if op == "append":
        B = _log(rng, 1, 256)
        T = B if rng.random() < 0.5 else max(B, min(_log(rng, B, 49152), MAX_TOKENS // (Hkv * (G + 2) * D)))
        layout = rng.choice(["half", "interleaved", "axis"])
        half = D // 2
        if layout == "axis":
            sections = rng.choice([(half,), (half // 2,) * 2, (half // 4,) * 3, (half // 4,) * 2])
        else:
            cut = half // 8 * rng.randint(2, 3)
            sections = rng.choice([(half,), (half // 2,), (half - cut, cut), (cut, (half - cut) // 2, (half - cut) // 2),
                                   (half // 4, half // 2 - half // 8, half // 2 - half // 8), (half // 3,) * 3])
        if layout == "half" and sum(sections) % 8:
            sections = (half,)
        held = min(rng.choice([0, _log(rng, 1, 1000), _log(rng, 1, 32768)]), MAX_HELD // (B * Hkv * D))
        return _drawn(_append("", B, T, Hkv * G, Hkv, D, page, sections, layout, rng.random() < 0.7, dtype, held))
    if op == "paged":
        B, N = _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 3, 5, 8])
        S = _log(rng, 1, 65536)
        S = max(1, min(S, MAX_KEYS // (B * Hkv * D)))
        return _drawn(_paged("", B, N, Hkv * G, Hkv, D, page, S, dtype, rng.random() < 0.8))
    B, S = _log(rng, 1, 64), _log(rng, 1, 4097)
    N = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 4097), _log(rng, 1, 31569)])
    N = max(1, min(N, 94707 // B, MAX_PAIRS // (B * S * Hkv * G * D)))
    return _drawn(_cross("", B, N, Hkv * G, Hkv, D, S, rng.choice(["equal", "ragged"]), dtype))


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _offsets(lens):
    got = [0]
    for n in lens:
        got.append(got[-1] + n)
    return got


def _split(r, total, parts):
    """`total` tokens in `parts` stretches of uneven lengths, none empty."""
    cuts = sorted(r.sample(range(1, total), parts - 1)) if parts > 1 else []
    return [b - a for a, b in zip([0, *cuts], [*cuts, total])]


def _append_plan(c):
    """Tokens held and new tokens of each request."""
    r = random.Random(c["B"] * 1009 + c["T"] * 31 + c["held"])
    held = [r.randint(0, c["held"]) for _ in range(c["B"])]
    return held, [1] * c["B"] if c["T"] == c["B"] else _split(r, c["T"], c["B"])


def _paged_plan(c):
    """Tokens held by each request, the new ones among them: ragged, the longest fills the cache; in a large
    batch one request has fewer than its new tokens, and one none."""
    r = random.Random(c["B"] * 7919 + c["S"])
    if not c["ragged"]:
        return [c["S"]] * c["B"]
    got = [r.randint(min(c["S"], c["N"]), c["S"]) for _ in range(c["B"])]
    got[0] = c["S"]
    if c["B"] > 8:
        got[3], got[6] = 0, min(c["S"], c["N"] // 2 + 1)
    return got


def _cross_plan(c):
    """Rows and encoder states of each sequence; in a large batch one has no encoder states."""
    r = random.Random(c["B"] * 3571 + c["N"] * 13 + c["S"])
    rows = [c["N"] if c["rows"] == "equal" else r.randint(1, c["N"]) for _ in range(c["B"])]
    states = [r.randint(1, c["S"]) for _ in range(c["B"])]
    rows[0], states[-1] = c["N"], c["S"]
    if c["B"] > 8:
        states[4] = 0
    return rows, states


def _table(c, counts, g):
    """Pages of each request, scattered over the cache; as many as `counts` tokens need, -1 behind them."""
    need = [-(-n // c["page"]) for n in counts]
    pages = sum(need) + 3  # a few that belong to nobody
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).tolist()
    width = max(max(need), 1)
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return pages, torch.tensor(rows, dtype=torch.int32, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _append_inputs(c, seed):
    g = _gen(seed)
    dt, D, Hq, Hkv, T = DTYPES[c["dtype"]], c["D"], c["Hq"], c["Hkv"], c["T"]
    held, new = _append_plan(c)
    pages, table = _table(c, [a + b for a, b in zip(held, new)], g)
    qkv = _randn(g, (T, Hq + 2 * Hkv, D), dt)  # as one projection leaves them
    s = {"q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + Hkv], "v": qkv[:, Hq + Hkv:], "table": table, "held": _ints(held),
         "offsets": None if T == c["B"] else _ints(_offsets(new)),
         "k_pages": _randn(g, (pages, c["page"], Hkv, D), dt), "v_pages": _randn(g, (pages, c["page"], Hkv, D), dt)}
    axes = c["sections"].count("-") + 1
    if axes > 1:  # (time, height, width) or (height, width); one axis: the place in the sequence
        s["positions"] = torch.stack([torch.randint(0, n, (T,), generator=g, device="cuda", dtype=torch.int32)
                                      for n in ((100000, 1000, 1000) if axes == 3 else (1000, 1000))], 1)
    if c["norm"]:
        s["q_weight"], s["k_weight"] = _randn(g, (D,), dt, 0.1, 1.0), _randn(g, (D,), dt, 0.1, 1.0)
    return s


def _paged_inputs(c, seed):
    g = _gen(seed)
    dt, D, Hkv = DTYPES[c["dtype"]], c["D"], c["Hkv"]
    lens = _paged_plan(c)
    pages, table = _table(c, lens, g)
    return {"q": _randn(g, (c["B"], c["N"], c["Hq"], D), dt), "table": table, "lengths": _ints(lens),
            "k_pages": _randn(g, (pages, c["page"], Hkv, D), dt), "v_pages": _randn(g, (pages, c["page"], Hkv, D), dt)}


def _cross_inputs(c, seed):
    g = _gen(seed)
    dt, D, Hkv = DTYPES[c["dtype"]], c["D"], c["Hkv"]
    rows, states = _cross_plan(c)
    kv = _randn(g, (sum(states), Hkv, 2 * D), dt)  # as one projection leaves them
    return {"q": _randn(g, (sum(rows), c["Hq"], D), dt), "k": kv[..., :D], "v": kv[..., D:],
            "q_offsets": None if c["rows"] == "equal" else _ints(_offsets(rows)), "k_offsets": _ints(_offsets(states))}


_INPUTS = {"append": _append_inputs, "paged": _paged_inputs, "cross": _cross_inputs}


def _sections(c):
    return tuple(int(n) for n in c["sections"].split("-"))


def prepare(case, seed):
    s = _INPUTS[case["op"]](case, seed)
    s["case"] = case
    if own:
        import __graft_entry__

        s["ops"] = __graft_entry__.load_package().ops
        if case["op"] == "append":  # the frequencies, laid out once as a model keeps them
            s["rope"] = s["ops"].RotaryAxes(case["D"], _sections(case), theta=10000.0, layout=case["layout"])
    elif case["op"] == "append":
        s["pairs"] = _pairs(case)
    return s


# -------------------------------------------------------------- plain forms
def _pairs(c):
    """Element of the first and of the second of each rotated pair, its axis and its frequency (64 bits)."""
    lo, hi, axis, freq = [], [], [], []
    total = sum(_sections(c))
    for a, n in enumerate(_sections(c)):
        for j in range(n):
            i = len(lo)
            if c["layout"] == "interleaved":
                lo.append(2 * i), hi.append(2 * i + 1)
            elif c["layout"] == "half":
                lo.append(i), hi.append(i + total)
            else:
                lo.append(2 * a * n + j), hi.append(2 * a * n + n + j)
            axis.append(a), freq.append(10000.0 ** (-j / n))
    return tuple(torch.tensor(t, device="cuda") for t in (lo, hi, axis)) + (
        torch.tensor(freq, dtype=torch.float64, device="cuda"),)


def _places(c, s):
    """Request of each token, its place there, and its row in the cache's pages."""
    T, B = c["T"], c["B"]
    token = torch.arange(T, device="cuda")
    if s["offsets"] is None:
        b = token // (T // B)
        start = b * (T // B)
    else:
        b = (token[:, None] >= s["offsets"][None, 1:]).sum(1)
        start = s["offsets"][b]
    place = s["held"][b] + token - start
    return place, s["table"][b, place // c["page"]].long() * c["page"] + place % c["page"]


def _plain_append(c, s):
    place, row = _places(c, s)
    lo, hi, axis, freq = s["pairs"]
    p = s["positions"] if "positions" in s else place[:, None]
    angle = p[:, axis].double() * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        y = x.clone()
        y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
        y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
        return y.to(s["q"].dtype)

    s["k_pages"].view(-1, c["Hkv"], c["D"])[row] = turned(s["k"], s.get("k_weight"))
    s["v_pages"].view(-1, c["Hkv"], c["D"])[row] = s["v"]
    return {"q": turned(s["q"], s.get("q_weight")), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_paged(c, s):
    B, N, H, G, D = c["B"], c["N"], c["Hkv"], c["Hq"] // c["Hkv"], c["D"]
    table = s["table"].long().clamp(min=0)
    k = s["k_pages"][table].flatten(1, 2).transpose(1, 2).float()  # [B, H, keys, D]
    v = s["v_pages"][table].flatten(1, 2).transpose(1, 2).float()
    q = s["q"].float().view(B, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * N, D) * D ** -0.5
    last = s["lengths"][:, None] - N + torch.arange(N, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") <= last[:, :, None]  # [B, N, keys]
    seen = seen[:, None, None].expand(B, 1, G, N, -1).reshape(B, 1, G * N, -1)
    score = torch.where(seen, q @ k.transpose(-1, -2), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    return o.view(B, H, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H * G, D).to(s["q"].dtype)


def _plain_cross(c, s):
    rows, states = map(_offsets, _cross_plan(c))
    G, D = c["Hq"] // c["Hkv"], c["D"]
    out = torch.empty_like(s["q"])
    for b in range(c["B"]):
        q = s["q"][rows[b]:rows[b + 1]].float().transpose(0, 1).unflatten(0, (-1, G)) * D ** -0.5  # [H, G, n, D]
        k = s["k"][states[b]:states[b + 1]].float().transpose(0, 1)[:, None]
        v = s["v"][states[b]:states[b + 1]].float().transpose(0, 1)[:, None]
        if states[b] == states[b + 1]:
            o = torch.zeros_like(q)
        else:
            score = q @ k.transpose(-1, -2)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = (p @ v) / p.sum(-1, keepdim=True)
        out[rows[b]:rows[b + 1]] = o.flatten(0, 1).transpose(0, 1).to(out.dtype)
    return out


_PLAIN = {"append": _plain_append, "paged": _plain_paged, "cross": _plain_cross}


def _own(c, s):
    ops = s["ops"]
    if c["op"] == "append":
        q = ops.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["held"],
                             offsets=s["offsets"], rope=s["rope"], positions=s.get("positions"),
                             q_weight=s.get("q_weight"), k_weight=s.get("k_weight"), eps=EPS)
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if c["op"] == "paged":
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"])
    return ops.cross_attention(s["q"], s["k"], s["v"], s["k_offsets"], q_offsets=s["q_offsets"])


def run(state):
    c = state["case"]
    return _own(c, state) if own else _PLAIN[c["op"]](c, state)


# ------------------------------------------------------------------- 64 bits
def _exact_append(c, s):
    held, new = _append_plan(c)
    secs = _sections(c)
    place = torch.cat([torch.arange(h, h + n, device="cuda") for h, n in zip(held, new)])
    req = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), torch.tensor(new, device="cuda"))
    pos = s["positions"].double() if "positions" in s else place.double()[:, None]
    turn = torch.cat([torch.outer(pos[:, a], 10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n))
                      for a, n in enumerate(secs)], 1)
    turn = torch.polar(torch.ones_like(turn), turn)[:, None]  # [T, 1, pairs]

    def head(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
        R = 2 * sum(secs)
        body, rest = x[..., :R], x[..., R:]
        if c["layout"] == "interleaved":
            z = torch.view_as_complex(body.unflatten(-1, (-1, 2)).contiguous()) * turn
            body = torch.view_as_real(z).flatten(-2)
        else:  # halves of the whole, or of each axis' own block
            blocks = body.unflatten(-1, (1 if c["layout"] == "half" else len(secs), 2, -1))
            z = torch.complex(blocks[..., 0, :].contiguous(), blocks[..., 1, :].contiguous())
            z = z * turn.view(-1, 1, *z.shape[2:])
            body = torch.stack([z.real, z.imag], -2).flatten(-3)
        return torch.cat([body, rest], -1)

    out = {"q": head(s["q"], s.get("q_weight"))}
    page = s["table"][req, torch.div(place, c["page"], rounding_mode="floor")].long()
    for name, val in (("k", head(s["k"], s.get("k_weight"))), ("v", s["v"].double())):
        out[name + "_pages"] = s[name + "_pages"].double()
        out[name + "_pages"][page, place % c["page"]] = val
    return out


def _exact_paged(c, s):
    N, G = c["N"], c["Hq"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_paged_plan(c)):
        ids = s["table"][b, :-(-n // c["page"])].long()
        k, v = (s[w][ids].flatten(0, 1)[:n].double() for w in ("k_pages", "v_pages"))  # [n, Hkv, D]
        for i in range(N):
            m = n - N + 1 + i  # keys that row i sees
            if m <= 0:
                continue
            q = s["q"][b, i].double().view(-1, G, c["D"])
            w = torch.einsum("hgd,shd->hgs", q, k[:m]) / math.sqrt(c["D"])
            out[b, i] = torch.einsum("hgs,shd->hgd", torch.softmax(w, -1), v[:m]).flatten(0, 1)
    return out


def _exact_cross(c, s):
    rows, states = _cross_plan(c)
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for q, o, k, v in zip(s["q"].split(rows), out.split(rows), s["k"].split(states), s["v"].split(states)):
        if k.shape[0]:
            for h in range(c["Hq"]):
                w = q[:, h].double() @ k[:, h // G].double().T / math.sqrt(c["D"])
                o[:, h] = torch.softmax(w, -1) @ v[:, h // G].double()
    return out


_EXACT = {"append": _exact_append, "paged": _exact_paged, "cross": _exact_cross}


def exact(case, seed):
    return _EXACT[case["op"]](case, _INPUTS[case["op"]](case, seed))


# ---------------------------------------------------------------------- work
def work(case):
    c = case
    D, Hq, Hkv = c["D"], c["Hq"], c["Hkv"]
    if c["op"] == "append":
        axes = c["sections"].count("-") + 1
        return {"bytes": c["T"] * ((2 * Hq + 4 * Hkv) * D * 2 + (4 * axes if axes > 1 else 0)),
                "flops": c["T"] * (Hq + Hkv) * D * (8 if c["norm"] else 4)}
    if c["op"] == "paged":
        lens = _paged_plan(c)
        seen = sum(max(0, n - c["N"] + 1 + i) for n in lens for i in range(c["N"]))
        return {"bytes": 4 * sum(lens) * Hkv * D + 4 * c["B"] * c["N"] * Hq * D, "flops": 4 * seen * Hq * D}
    rows, states = _cross_plan(c)
    return {"bytes": 4 * sum(states) * Hkv * D + 4 * sum(rows) * Hq * D,
            "flops": 4 * sum(a * b for a, b in zip(rows, states)) * Hq * D}
