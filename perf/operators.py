"""Operators on weights and caches held in 4 bits: what is measured, their plain forms, and the calls of the framework.

    listed()            the cases that are measured
    draw(rng)           another case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the plain form, or with `own` the framework's kernels
    exact(case, seed)   what `run` returns, computed in 64 bits
    work(case)          bytes and operations that a pass cannot do without

linear     y = act(a W^T), W[n, k] = s[n, k / group] (q[n, k] - 8): plain, or gated with rows that alternate eight gates, eight ups
experts    router's choice, gated and plain products of the chosen experts, weighted sum, norm and residual
attention  the step's positions are appended to a cache of 4-bit keys and values, then every row attends over what it may see
"""
import ctypes as C
import math
import zlib

import torch

own = False

DEV = "cuda"
GRAPH_ROWS = 128      # up to here a product is replayed as a graph, as a decode step is
EPS = 1e-5


def listed():
    return [
        # one token's output projection: the smallest call, where launches count
        {"name": "linear 1 row 4096x4096", "kind": "linear", "m": 1, "k": 4096, "n": 4096, "group": 128, "act": "none", "out": "float32"},
        # sixteen sequences decoding through a wide gated feed-forward
        {"name": "linear 16 rows gated 4096x28672", "kind": "linear", "m": 16, "k": 4096, "n": 28672, "group": 64, "act": "swish", "out": "bfloat16"},
        # three sequences through the long K of `down`, small groups
        {"name": "linear 3 rows 14336x4096", "kind": "linear", "m": 3, "k": 14336, "n": 4096, "group": 32, "act": "none", "out": "float32"},
        # a ragged portion of a prompt together with decoding sequences
        {"name": "linear 100 rows 4096x14330", "kind": "linear", "m": 100, "k": 4096, "n": 14330, "group": 128, "act": "none", "out": "float32"},
        # a prompt
        {"name": "linear 2048 rows gated 4096x28672", "kind": "linear", "m": 2048, "k": 4096, "n": 28672, "group": 128, "act": "gelu", "out": "bfloat16"},
        # a few sequences decoding through a layer of experts
        {"name": "experts 5 tokens", "kind": "experts", "m": 5, "width": 2048, "ff": 1024, "experts": 64, "identity": 16, "top": 8, "groups": 8, "keep": 4,
         "group": 64},
        # a ragged prompt through the same layer
        {"name": "experts 777 tokens", "kind": "experts", "m": 777, "width": 2048, "ff": 1024, "experts": 64, "identity": 16, "top": 8, "groups": 8, "keep": 4,
         "group": 64},
        # one sequence decoding
        {"name": "attention 1 token at 2000", "kind": "attention", "seqs": 1, "tokens": 1, "context": 2000, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "slopes": False, "sink": True},
        # sixteen sequences decoding, of different lengths
        {"name": "attention 16 x 1 at 4096", "kind": "attention", "seqs": 16, "tokens": 1, "context": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "slopes": True, "sink": False},
        # four long sequences decoding
        {"name": "attention 4 x 1 at 60000", "kind": "attention", "seqs": 4, "tokens": 1, "context": 60000, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "slopes": False, "sink": True},
        # a few tokens of three sequences at once, narrow heads, odd lengths
        {"name": "attention 3 x 5 at 7001", "kind": "attention", "seqs": 3, "tokens": 5, "context": 7001, "heads": 16, "kv_heads": 4, "dim": 64, "vdim": 64,
         "slopes": False, "sink": True},
        # a portion of a prompt behind a cached one
        {"name": "attention 1 x 2000 at 1000", "kind": "attention", "seqs": 1, "tokens": 2000, "context": 1000, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "slopes": False, "sink": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "attention", "attention"])
    if kind == "linear":
        act, group = rng.choice(["none", "none", "gelu", "swish"]), rng.choice([32, 64, 128])
        k, n = 128 * _log_int(rng, 4, 112), _log_int(rng, 200, 28000)
        m = _log_int(rng, 1, max(1, min(2000, 2048 * 4096 * 28672 // (k * n))))
        if act != "none":
            n = max(16, n // 16 * 16)
        return {"kind": kind, "m": m, "k": k, "n": n, "group": group, "act": act, "out": rng.choice(["float32", "bfloat16"]) if act == "none" else "bfloat16"}
    if kind == "experts":
        groups = rng.choice([1, 4, 8])
        return {"kind": kind, "m": _log_int(rng, 1, 770), "width": 128 * rng.randrange(4, 17), "ff": 64 * rng.randrange(4, 17), "experts": 8 * rng.randrange(2, 9),
                "identity": rng.choice([0, 8, 16]), "top": rng.randrange(1, 9), "groups": groups, "keep": max(1, groups // 2), "group": rng.choice([32, 64])}
    mode = rng.choice(["decode", "decode", "few", "prompt"])
    kv = rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "heads": kv * rng.choice([1, 2, 4, 8]), "kv_heads": kv, "dim": rng.choice([64, 80, 128]), "vdim": rng.choice([64, 96, 128]),
            "slopes": rng.random() < 0.5, "sink": rng.random() < 0.5}
    if mode == "decode":
        case.update(seqs=_log_int(rng, 1, 32), tokens=1)
        case["context"] = _log_int(rng, 10, max(20, min(60000, 240000 // case["seqs"])))
    elif mode == "few":
        case.update(seqs=rng.randrange(1, 9), tokens=rng.randrange(2, 17), context=_log_int(rng, 10, 16000))
    else:
        case.update(seqs=rng.randrange(1, 3), tokens=_log_int(rng, 20, 1500), context=_log_int(rng, 1, 2000))
    # no more scores than the listed portion of a prompt has
    while case["seqs"] * case["tokens"] * case["heads"] * (case["context"] + case["tokens"]) > 2000 * 32 * 1500:
        case["context"], case["tokens"] = (case["context"] + 1) // 2, (case["tokens"] + 1) // 2
    return case


def _gen(seed, name):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + zlib.crc32(name.encode())) % (1 << 62))


def _randn(seed, name, *shape):
    return torch.randn(*shape, generator=_gen(seed, name), device=DEV)


# ---- numbers of 4 bits --------------------------------------------------------------------------------------------
def _quantise(v, group):
    """f32 [..., K] -> quants 0 .. 15 [..., K] and bf16 scales [..., K / group]: the value of largest magnitude (the first of equals) is -8 steps."""
    v = v.unflatten(-1, (-1, group))
    a = v.abs()
    first = (a == a.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
    s = (v.gather(-1, first)[..., 0] / -8.0).bfloat16()
    d = s.float()[..., None]
    q = torch.where(d == 0, torch.full_like(v, 8.0), (torch.round(v / torch.where(d == 0, torch.ones_like(d), d)) + 8.0).clamp(0, 15))
    return q.flatten(-2).to(torch.uint8), s


def _values(q, s, group, dtype=torch.float32):
    return ((q.to(dtype) - 8.0).unflatten(-1, (-1, group)) * s.to(dtype)[..., None]).flatten(-2)


def _packed(q):
    """Two quants a byte, the first in the low half."""
    return q[..., 0::2] | (q[..., 1::2] << 4)


def _unpacked(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


# ---- linears ------------------------------------------------------------------------------------------------------
def _gated(y, act, limit):
    """Columns that alternate eight gates, eight ups -> gated columns."""
    y = y.unflatten(-1, (-1, 2, 8))
    g, u = y[..., 0, :].flatten(-2), y[..., 1, :].flatten(-2)
    if act == "gelu":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g / (1.0 + torch.exp(-1.702 * g)) * (u + 1.0)


LIMIT = 7.0


def _linear_inputs(case, seed):
    m, k, n = case["m"], case["k"], case["n"]
    a = _randn(seed, "a", m, k)
    # decoding meets channels that stand out
    a[:, torch.rand(k, generator=_gen(seed, "channels"), device=DEV) < 0.01] *= 20.0
    q, s = _quantise(_randn(seed, "w", n, k) * 0.02, case["group"])
    return a.bfloat16(), _packed(q), s


def _prepare_linear(case, seed):
    a, q, s = _linear_inputs(case, seed)
    state = {"case": case, "a": a, "q": q, "s": s, "out": getattr(torch, case["out"])}
    if own:
        state["plan"] = OwnLinear(state)
    return state


def _linear_plain(a, q, s, case, dtype=torch.float32):
    y = a.to(dtype) @ _values(_unpacked(q), s, case["group"], dtype).t()
    return y if case["act"] == "none" else _gated(y, case["act"], LIMIT)


def _run_linear(state):
    if own:
        return state["plan"].run()
    return _linear_plain(state["a"], state["q"], state["s"], state["case"]).to(state["out"])


def _exact_linear(case, seed):
    a, q, s = _linear_inputs(case, seed)
    w = (torch.stack([q & 15, q >> 4], -1).view(case["n"], -1, case["group"]).double() - 8.0) * s.double().unsqueeze(2)
    y = torch.nn.functional.linear(a.double(), w.view(case["n"], case["k"]))
    if case["act"] == "none":
        return y
    y = y.view(case["m"], -1, 2, 8)
    g, u = y[:, :, 0].reshape(case["m"], -1), y[:, :, 1].reshape(case["m"], -1)
    if case["act"] == "gelu":
        return torch.nn.functional.gelu(g, approximate="tanh") * u
    g, u = torch.clamp(g, max=LIMIT), torch.clamp(u, -LIMIT, LIMIT)
    return g * torch.sigmoid(1.702 * g) * (u + 1.0)


# ---- a layer of experts -------------------------------------------------------------------------------------------
def _expert_inputs(case, seed):
    m, N, F, E, g = case["m"], case["width"], case["ff"], case["experts"], case["group"]
    every = E + case["identity"]
    x = _randn(seed, "x", m, N)
    both = _quantise(_randn(seed, "gate_up", E, 2 * F, N) * N ** -0.5, g)
    down = _quantise(_randn(seed, "down", E, N, F) * F ** -0.5, g)
    return {"x": x, "h": x.bfloat16(), "logits": _randn(seed, "logits", m, every) * 1.5, "correction": _randn(seed, "correction", every) * 0.01,
            "both": (_packed(both[0]), both[1]), "down": (_packed(down[0]), down[1]), "norm": 1.0 + 0.1 * _randn(seed, "norm", N),
            "scale": 0.5 + 0.1 * _randn(seed, "scale", N)}


def _prepare_experts(case, seed):
    state = {"case": case, **_expert_inputs(case, seed)}
    if own:
        state["plan"] = OwnExperts(state)
    return state


def _chosen(logits, correction, case):
    """Weights [m, experts + identity]: the softmax scores of the chosen outputs, zero elsewhere."""
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    c = p + correction.to(p.dtype)
    if case["groups"] > 1:
        best = c.unflatten(-1, (case["groups"], -1)).amax(-1)
        ok = torch.zeros_like(best, dtype=torch.bool).scatter_(1, best.topk(case["keep"], -1).indices, True)
        c = c.masked_fill(~ok.repeat_interleave(c.shape[1] // case["groups"], 1), -math.inf)
    at = c.topk(case["top"], -1).indices
    return torch.zeros_like(p).scatter_(1, at, p.gather(1, at))


def _experts_plain(s, dtype):
    case = s["case"]
    E, g = case["experts"], case["group"]
    w = _chosen(s["logits"].to(dtype), s["correction"], case)
    a = torch.einsum("mk,enk->men", s["h"].to(dtype), _values(_unpacked(s["both"][0]), s["both"][1], g, dtype))
    a = _gated(a, "swish", LIMIT) * w[:, :E, None]
    y = torch.einsum("mef,enf->mn", a, _values(_unpacked(s["down"][0]), s["down"][1], g, dtype))
    x = s["x"].to(dtype)
    y = y + x * w[:, E:].sum(-1, keepdim=True)
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * s["norm"].to(dtype)
    return x + s["scale"].to(dtype) * y


def _run_experts(state):
    if own:
        return state["plan"].run()
    return _experts_plain(state, torch.float32).bfloat16()


def _exact_experts(case, seed):
    s = _expert_inputs(case, seed)
    E, F, N, g = case["experts"], case["ff"], case["width"], case["group"]
    p = torch.softmax(s["logits"].double(), -1)
    c = p + s["correction"].double()
    if case["groups"] > 1:
        parts = c.view(case["m"], case["groups"], -1)
        rank = parts.amax(2).argsort(1, descending=True).argsort(1)
        c = torch.where((rank < case["keep"])[:, :, None], parts, torch.full_like(parts, -math.inf)).view_as(c)
    keep = c.argsort(1, descending=True).argsort(1) < case["top"]
    w = torch.where(keep, p, torch.zeros_like(p))
    x, h = s["x"].double(), s["h"].double()
    y = x * w[:, E:].sum(1, keepdim=True)
    for e in range(E):
        t = w[:, e].nonzero()[:, 0]
        if not len(t):
            continue
        mat = [((torch.stack([b[e] & 15, b[e] >> 4], -1).view(rows, -1, g).double() - 8.0) * sc[e].double()[:, :, None]).view(rows, -1)
               for (b, sc), rows in ((s["both"], 2 * F), (s["down"], N))]
        z = (h[t] @ mat[0].t()).view(len(t), -1, 2, 8)
        gate, up = z[:, :, 0].reshape(len(t), F).clamp(max=LIMIT), z[:, :, 1].reshape(len(t), F).clamp(-LIMIT, LIMIT)
        y[t] += w[t, e, None] * ((gate * torch.sigmoid(1.702 * gate) * (up + 1.0)) @ mat[1].t())
    return x + s["scale"].double() * (y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * s["norm"].double())


# ---- attention ----------------------------------------------------------------------------------------------------
# A head's part of a cache comes in tiles of 16 positions: the quants of 32 columns after those of 32 columns, 256 bytes each, then for the pairs of
# positions the scales of every 32 columns, both positions side by side.  How the quants of a tile lie:
#   keys    position 8 n + r, column 16 s + 4 t + 2 i + h -> byte [r][t][s][2 h + n], low half for i = 0
#   values  position 8 i + 2 t + h, column 16 s + 8 n + r -> byte [r][t][s][2 h + i], low half for n = 0
def _up(v, to):
    return (v + to - 1) // to * to


def _to_tiles(q, s, values):
    """Quants [..., P, W] and scales [..., P, W / 32] (P a multiple of 16) -> bytes [..., P / 16, tile]."""
    lead, P, W = q.shape[:-2], q.shape[-2], q.shape[-1]
    n = len(lead)
    base = list(range(n + 1))
    if values:
        q = q.view(*lead, P // 16, 2, 4, 2, W // 32, 2, 2, 8)              # tile, i, t, h, group, s, n, r
        q = q.permute(*base, n + 4, n + 7, n + 2, n + 5, n + 3, n + 1, n + 6)  # tile, group, r, t, s, h, i, n
    else:
        q = q.view(*lead, P // 16, 2, 8, W // 32, 2, 4, 2, 2)              # tile, n, r, group, s, t, i, h
        q = q.permute(*base, n + 3, n + 2, n + 5, n + 4, n + 7, n + 1, n + 6)  # tile, group, r, t, s, h, n, i
    b = (q[..., 0] | (q[..., 1] << 4)).reshape(*lead, P // 16, W // 32 * 256)
    sc = s.view(*lead, P // 16, 8, 2, W // 32).transpose(-1, -2).contiguous().view(torch.uint8).reshape(*lead, P // 16, W // 32 * 32)
    return torch.cat([b, sc], -1).contiguous()


def _from_tiles(b, values):
    """Bytes [..., P / 16, tile] -> quants [..., P, W] and scales [..., P, W / 32]."""
    lead, T = b.shape[:-2], b.shape[-2]
    W = b.shape[-1] // 288 * 32
    n = len(lead)
    base = list(range(n + 1))
    q = b[..., :W * 8].reshape(*lead, T, W // 32, 8, 4, 2, 2, 2)           # tile, group, r, t, s, h, n (i)
    q = torch.stack([q & 15, q >> 4], -1)                                  # ..., i (n)
    if values:
        q = q.permute(*base, n + 6, n + 3, n + 5, n + 1, n + 4, n + 7, n + 2)  # i, t, h, group, s, n, r
    else:
        q = q.permute(*base, n + 6, n + 2, n + 1, n + 4, n + 3, n + 7, n + 5)  # n, r, group, s, t, i, h
    s = b[..., W * 8:].contiguous().view(torch.bfloat16).view(*lead, T, 8, W // 32, 2).transpose(-1, -2)
    return q.reshape(*lead, T * 16, W), s.reshape(*lead, T * 16, W // 32)


def _cache_values(b, values, width, dtype=torch.float32):
    q, s = _from_tiles(b, values)
    return _values(q, s, 32, dtype)[..., :width]


def _pad32(v):
    return torch.nn.functional.pad(v, (0, _up(v.shape[-1], 32) - v.shape[-1]))


def _attention_inputs(case, seed):
    S, T, H, G, D, V, ctx = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "vdim", "context"))
    cap = _up(ctx + T, 16)
    # sequences of different lengths, the first the longest
    pos0 = ctx - (torch.rand(S, generator=_gen(seed, "lengths"), device=DEV) * (ctx // 2)).to(torch.int32)
    pos0[0] = ctx
    q, k, v = _randn(seed, "q", S * T, H * D) * 1.5, _randn(seed, "k", S * T, G * D), _randn(seed, "v", S * T, G * V)
    # some columns of the keys stand out
    loud = 1.0 + 4.0 * (torch.rand(G * D, generator=_gen(seed, "loud"), device=DEV) < 0.03)
    k *= loud
    kc = _to_tiles(*_quantise(_pad32(_randn(seed, "kc", S, G, cap, D) * loud.view(G, 1, D)), 32), False)
    vc = _to_tiles(*_quantise(_pad32(_randn(seed, "vc", S, G, cap, V)), 32), True)
    return {"pos0": pos0, "proj": torch.cat([q, k, v], -1), "kc": kc, "vc": vc, "cap": cap,
            "slopes": torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H).float() if case["slopes"] else None}


def _prepare_attention(case, seed):
    state = {"case": case, **_attention_inputs(case, seed)}
    S, T = case["seqs"], case["tokens"]
    state["pos"] = (state["pos0"][:, None] + torch.arange(T, device=DEV, dtype=torch.int32)).contiguous()
    if own:
        state["plan"] = OwnAttention(state)
    return state


def _split(state):
    case = state["case"]
    S, T, H, G, D, V = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "vdim"))
    q, k, v = state["proj"].split([H * D, G * D, G * V], -1)
    return q.view(S, T, G, H // G, D), k.view(S, T, G, D), v.view(S, T, G, V)


def _append(cache, values, rows, at):
    """The cache's tiles with the step's rows [S, T, G, W] at positions `at` [S, T]."""
    q, s = _from_tiles(cache, values)
    nq, ns = _quantise(_pad32(rows), 32)
    idx = at.long()[:, None, :, None]
    q = q.scatter(2, idx.expand(-1, q.shape[1], -1, q.shape[3]), nq.transpose(1, 2))
    s = s.scatter(2, idx.expand(-1, s.shape[1], -1, s.shape[3]), ns.transpose(1, 2))
    return _to_tiles(q, s, values), _values(q, s, 32)


def _run_attention(state):
    if own:
        return state["plan"].run()
    case = state["case"]
    S, T, H, G, D, V = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "vdim"))
    q, k, v = _split(state)
    kc, keys = _append(state["kc"], False, k, state["pos"])
    vc, vals = _append(state["vc"], True, v, state["pos"])
    state["kc"].copy_(kc), state["vc"].copy_(vc)
    z = torch.einsum("stgrd,sgpd->sgrtp", q, keys[..., :D]) * D ** -0.5
    back = (state["pos"][:, :, None] - torch.arange(z.shape[-1], device=DEV))[:, None, None]
    if state["slopes"] is not None:
        z = z - state["slopes"].view(1, G, H // G, 1, 1) * back
    z = z.masked_fill(back < 0, -math.inf)
    top = z.amax(-1, keepdim=True)
    if case["sink"]:
        top = top.clamp(min=0.0)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True) + (torch.exp(-top) if case["sink"] else 0.0)
    o = torch.einsum("sgrtp,sgpv->stgrv", p / total, vals[..., :V])
    return {"out": o.reshape(S * T, H * V).bfloat16(), "keys": state["kc"], "values": state["vc"]}


def _exact_attention(case, seed):
    s = _attention_inputs(case, seed)
    S, T, H, G, D, V = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "vdim"))
    q, k, v = s["proj"].split([H * D, G * D, G * V], -1)
    out = torch.empty(S, T, H, V, dtype=torch.float64, device=DEV)
    new = [_values(*_quantise(_pad32(x.view(S, T, G, -1)), 32), 32, torch.float64) for x in (k, v)]
    for i in range(S):
        p0 = int(s["pos0"][i])
        for g in range(G):
            K, Vv = (torch.cat([_cache_values(c[i, g], val, w, torch.float64)[:p0], n[i, :, g, :w]]) for c, val, w, n in
                     ((s["kc"], False, D, new[0]), (s["vc"], True, V, new[1])))
            back = torch.arange(p0, p0 + T, device=DEV)[:, None] - torch.arange(p0 + T, device=DEV)
            for h in range(g * (H // G), (g + 1) * (H // G)):
                z = q.view(S, T, H, D)[i, :, h].double() @ K.t() / math.sqrt(D)
                if s["slopes"] is not None:
                    z = z - s["slopes"][h].double() * back
                z = torch.where(back < 0, torch.full_like(z, -math.inf), z)
                if case["sink"]:
                    z = torch.cat([z, torch.zeros(T, 1, dtype=torch.float64, device=DEV)], 1)
                out[i, :, h] = torch.softmax(z, 1)[:, :p0 + T] @ Vv
    return {"out": out.view(S * T, H * V), "keys": None, "values": None}


# ---- the framework's calls ----------------------------------------------------------------------------------------
_contexts = {}


def _context():
    """A context of the language models' library on a stream that torch shares."""
    if "lm" not in _contexts:
        from peregrine_b200.runtime import GpuContext

        stream = torch.cuda.Stream()
        _contexts["lm"] = (GpuContext(0, stream.cuda_stream, "lm"), stream)
    return _contexts["lm"]


def _device(rows):
    from peregrine_b200.layers import Device

    return Device(_context()[0], "bfloat16", rows)


class Recorded:
    """A call, replayed as a graph where it is a decode step's."""

    def record(self):
        gpu = _context()[0]
        torch.cuda.synchronize()
        self.call()
        gpu.sync()
        with gpu.record() as g:
            self.call()
        self.graph = g

    def run(self):
        if self.graph is not None:
            self.graph.launch()
        else:
            self.call()
        return self.result

    def __del__(self):
        torch.cuda.synchronize()
        if getattr(self, "graph", None) is not None:
            self.graph.free()
        self.free()


class OwnLinear(Recorded):
    def __init__(self, state):
        from peregrine_b200 import _lib
        from peregrine_b200.layers import Linear4

        case = state["case"]
        self.d = _device(case["m"])
        self.a = state["a"]
        torch.cuda.synchronize()
        self.w = Linear4.from_quants(self.d, state["q"], state["s"])
        self.act = {"none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU_TANH_GLU, "swish": _lib.ACT_CLAMPED_SWISH_GLU}[case["act"]]
        cols = case["n"] if case["act"] == "none" else case["n"] // 2
        # rows of bf16 outputs start on 16-byte boundaries
        self.y = torch.zeros(case["m"], _up(cols, 8), dtype=state["out"], device=DEV)
        self.m, self.result, self.graph = case["m"], self.y[:, :cols], None
        if self.m <= GRAPH_ROWS:
            self.record()

    def call(self):
        self.w.run(self.a, self.m, self.y, self.act, LIMIT)

    def free(self):
        self.w.free()


class OwnExperts(Recorded):
    def __init__(self, state):
        from peregrine_b200.layers import Linear4

        case = self.case = state["case"]
        self.gpu, self.stream = _context()
        d = self.d = _device(case["m"])
        torch.cuda.synchronize()
        self.s = state
        self.both, self.down = Linear4.from_quants(d, *state["both"]), Linear4.from_quants(d, *state["down"])
        self.route = C.c_void_p()
        d.check(d.lib.pg_route_create(self.gpu.handle, case["m"], case["experts"], case["identity"], case["top"], C.byref(self.route)))
        rows = int(d.lib.pg_route_max_rows(self.route))
        self.mid = torch.zeros(rows, _up(case["ff"], 64), dtype=torch.bfloat16, device=DEV)
        self.outs = torch.zeros(rows, case["width"], dtype=torch.bfloat16, device=DEV)
        self.x = torch.zeros_like(state["x"])
        self.result, self.graph = torch.zeros_like(state["h"]), None
        if case["m"] <= GRAPH_ROWS:
            self.record()

    def call(self):
        from peregrine_b200 import _lib

        d, c, s, h = self.d, self.case, self.s, self.gpu.handle
        lib, m, N = d.lib, c["m"], c["width"]
        with torch.cuda.stream(self.stream):
            self.x.copy_(s["x"])
        d.check(lib.pg_route_run(h, self.route, d.code, s["logits"].data_ptr(), s["logits"].stride(0), m, s["correction"].data_ptr(), c["groups"], c["keep"]))
        self.both.run_routed(self.route, s["h"], True, self.mid, _lib.ACT_CLAMPED_SWISH_GLU, LIMIT)
        self.down.run_routed(self.route, self.mid, False, self.outs)
        d.check(lib.pg_routed_norm_add(h, self.route, self.outs.data_ptr(), self.outs.stride(0), self.x.data_ptr(), s["norm"].data_ptr(), s["scale"].data_ptr(), m,
                                       N, EPS, self.result.data_ptr(), d.code, self.result.stride(0)))

    def free(self):
        self.both.free()
        self.down.free()
        self.d.lib.pg_route_free(self.gpu.handle, self.route)


class OwnAttention(Recorded):
    def __init__(self, state):
        from peregrine_b200.layers import Attention4Plan, Batch

        case = state["case"]
        S, T, H, G, D, V = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "vdim"))
        self.d = _device(S * T)
        self.s = state
        self.out = torch.zeros(S * T, H * V, dtype=torch.bfloat16, device=DEV)
        self.plan = Attention4Plan(self.d, H, G, D, V, state["cap"], S, S, scale=D ** -0.5, sink=case["sink"], slopes=state["slopes"])
        self.batch = Batch(self.d, [(i, p, [0] * T) for i, p in enumerate(state["pos0"].tolist())], fixed=True)
        self.result, self.graph = {"out": self.out, "keys": state["kc"], "values": state["vc"]}, None
        if S * T <= GRAPH_ROWS:
            self.record()

    def call(self):
        self.plan.run(self.batch, self.s["proj"], self.s["kc"], self.s["vc"], self.out)

    def free(self):
        self.plan.free()


# ---- the interface ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    return {"linear": _prepare_linear, "experts": _prepare_experts, "attention": _prepare_attention}[case["kind"]](case, seed)


def run(state):
    return {"linear": _run_linear, "experts": _run_experts, "attention": _run_attention}[state["case"]["kind"]](state)


def exact(case, seed):
    return {"linear": _exact_linear, "experts": _exact_experts, "attention": _exact_attention}[case["kind"]](case, seed)


def work(case):
    if case["kind"] == "linear":
        m, k, n, g = (case[x] for x in ("m", "k", "n", "group"))
        cols = n if case["act"] == "none" else n // 2
        return {"bytes": n * k // 2 + 2 * n * (k // g) + 2 * m * k + m * cols * (4 if case["out"] == "float32" else 2), "flops": 2 * m * k * n}
    if case["kind"] == "experts":
        m, N, F, E, g = (case[x] for x in ("m", "width", "ff", "experts", "group"))
        every = E + case["identity"]
        used = E * (1.0 - (1.0 - case["top"] / every) ** m)
        pairs = m * case["top"] * E / every
        return {"bytes": used * 3 * N * F * (0.5 + 2.0 / g) + m * (4 * every + 4 * N + 2 * N + 2 * N), "flops": 6.0 * N * F * pairs}
    S, T, H, G, D, V, ctx = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "vdim", "context"))
    held = (ctx + (S - 1) * (ctx - ctx / 4)) + S * T              # positions read, of sequences between half and the whole context
    seen = (held - S * T) * T + S * T * (T + 1) / 2
    return {"bytes": held * G * (D + V) * 0.5625 + S * T * (4 * (H * D + G * (D + V)) + 2 * H * V), "flops": 2.0 * seen * H * (D + V)}
