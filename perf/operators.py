"""Speculative decoding's operators as cases that can be timed and checked: rotating and storing a pass's queries and keys,
attention of a tree of drafted tokens over the KV cache, log probabilities of the drafted tokens, and moving the accepted
tokens' cache rows to their places (or a whole prefix into another cache).

Each case is one call. Where `own` is false, `run` is the operator's formula in elementary torch operations; where it is
true, the call of webllm_amd.qlinear that computes it, on inputs that lie in the library's arenas. `exact` is the same in
64-bit arithmetic.
"""
import math

import torch

own = False

# (heads, kv heads, head dim, layers) of the two model shapes that the benchmark and the tests use.
MODELS = {"05b": (14, 2, 64, 24), "7b": (28, 4, 128, 28)}
THETA = 1e6
EPS = 1e-6
VOCAB = 151936


def listed():
    return [
        # One decoded token of the small model: its 14 query and 2 key heads rotated, key and value stored. Launch latency.
        {"name": "rope_05b_m1", "kind": "rope", "model": "05b", "M": 1, "pos": 500, "cache": "f32", "norm": False,
         "rot": 64, "interleaved": False, "fused": False},
        # A drafted tree of 24 tokens far into a context: q, k and v from one projection's rows, heads normed, a half cache.
        {"name": "rope_7b_m24", "kind": "rope", "model": "7b", "M": 24, "pos": 30000, "cache": "f16", "norm": True,
         "rot": 128, "interleaved": False, "fused": True},
        # A prompt of 2048 tokens, heads normed: a stream through memory.
        {"name": "rope_7b_m2048", "kind": "rope", "model": "7b", "M": 2048, "pos": 0, "cache": "f32", "norm": True,
         "rot": 128, "interleaved": False, "fused": False},
        # Five drafted tokens early in a chat: latency.
        {"name": "tree_05b_m5_t300", "kind": "tree", "model": "05b", "M": 5, "past": 300, "cache": "f32", "chain": False},
        # A single token over a long half cache: the cache is read once, memory-bound.
        {"name": "tree_7b_m1_t32000", "kind": "tree", "model": "7b", "M": 1, "past": 32000, "cache": "f16", "chain": False},
        # An ordinary drafted tree at an ordinary context.
        {"name": "tree_7b_m24_t4000", "kind": "tree", "model": "7b", "M": 24, "past": 4000, "cache": "f32", "chain": False},
        # The largest tree over a long half cache: matrix-core bound. (A chain: also a prompt's chunk over such a cache.)
        {"name": "tree_7b_m256_t8000", "kind": "tree", "model": "7b", "M": 256, "past": 8000, "cache": "f16", "chain": True},
        # The sampled token's log probability with the five best alternatives, as an API returns them.
        {"name": "logprobs_m1", "kind": "logprobs", "M": 1, "V": VOCAB, "T": 1, "top": 5, "masked": False},
        # Verification of a drafted tree: up to four children per node and 20 alternatives, under a grammar's mask.
        {"name": "logprobs_m24", "kind": "logprobs", "M": 24, "V": VOCAB, "T": 4, "top": 20, "masked": True},
        # Scoring of a 512-token text: every row of the logits read once.
        {"name": "logprobs_m512", "kind": "logprobs", "M": 512, "V": VOCAB, "T": 1, "top": 0, "masked": False},
        # Four accepted tokens of a tree of 24 moved to the end of the context, in every layer's cache.
        {"name": "move_05b_accept", "kind": "move", "model": "05b", "cache": "f32", "n": 4, "rows": 24, "past": 300},
        # A prompt of 2000 tokens copied into another sequence's cache.
        {"name": "move_7b_fork", "kind": "move", "model": "7b", "cache": "f16", "n": 2000, "rows": 0, "past": 0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "tree", "tree", "logprobs", "logprobs", "move"])
    model, cache = rng.choice(["05b", "7b"]), rng.choice(["f32", "f16"])
    D = MODELS[model][2]
    if kind == "rope":
        return {"kind": kind, "model": model, "M": _log(rng, 1, 2048), "pos": _log(rng, 1, 100000), "cache": cache,
                "norm": rng.random() < 0.5, "rot": rng.choice([D, D, D // 2]), "interleaved": rng.random() < 0.3,
                "fused": rng.random() < 0.4}
    if kind == "tree":
        M, past = _log(rng, 1, 256), 0 if rng.random() < 0.1 else _log(rng, 16, 32000)
        while M * (past + M) > 256 * 8200:
            past //= 2
        return {"kind": kind, "model": model, "M": M, "past": past, "cache": cache, "chain": rng.random() < 0.3}
    if kind == "logprobs":
        V = VOCAB if rng.random() < 0.6 else _log(rng, 50, 160000)
        M = _log(rng, 1, max(2, min(1024, 512 * VOCAB // V)))
        return {"kind": kind, "M": M, "V": V, "T": rng.randint(0, 6), "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                "masked": rng.random() < 0.3}
    if rng.random() < 0.5:
        n = _log(rng, 1, 16)
        return {"kind": kind, "model": model, "cache": cache, "n": n, "rows": n + _log(rng, 1, 100), "past": _log(rng, 1, 2000)}
    n = _log(rng, 20, 1000 if cache == "f32" else 2000)
    return {"kind": kind, "model": model, "cache": cache, "n": n, "rows": 0, "past": 0}


# ------------------------------------------------------------------ inputs, from the seed alone

_TYPES = {"f32": torch.float32, "f16": torch.float16}
_BYTES = {"f32": 4, "f16": 2}


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _parents(g, M, chain):
    """A tree in breadth-first order: each token continues an earlier one, or (-1) the context."""
    if chain:
        return torch.arange(-1, M - 1, device="cuda")
    at = torch.arange(M, device="cuda")
    return (torch.rand(M, generator=g, device="cuda") * (at + 1) * 0.9).floor().long() - 1


def _ancestors(parents):
    """[M, M]: whether token j is token m or one that it continues: the inverse of I - (m's parent is j), whole numbers."""
    M = parents.numel()
    step = torch.zeros(M, M + 1, dtype=torch.float64, device="cuda").scatter_(1, (parents % (M + 1))[:, None], 1.0)[:, :M]
    eye = torch.eye(M, dtype=torch.float64, device="cuda")
    return torch.linalg.solve_triangular(eye - step, eye, upper=False, unitriangular=True) > 0.5


def _words(seen):
    """[M, ceil(M / 64)] int64: bit j % 64 of word j / 64 tells whether column j is seen."""
    M = seen.shape[0]
    wide = torch.nn.functional.pad(seen, (0, -M % 64)).reshape(M, -1, 64).long()
    return (wide << torch.arange(64, device="cuda")).sum(-1)


def _inputs(case, seed):
    g, kind = torch.Generator(device="cuda").manual_seed(int(seed)), case["kind"]
    if kind == "logprobs":
        M, V = case["M"], case["V"]
        x = _normal(g, M, V, scale=2.5)
        x[torch.arange(M, device="cuda")[:, None], torch.randint(V, (M, 3), generator=g, device="cuda")] += 12.0
        if case["masked"]:
            keep = torch.rand(M, V, generator=g, device="cuda") < max(0.01, 8 / V)
            if M > 1:
                keep[-1] = False                                                     # a row with nothing allowed
            x = torch.where(keep, x, -math.inf)
        tokens = torch.randint(V, (M, case["T"]), generator=g, device="cuda", dtype=torch.int32)
        tokens[:, 1:][torch.rand(M, max(0, case["T"] - 1), generator=g, device="cuda") < 0.3] = -1    # fewer children
        return {"logits": x, "tokens": tokens}
    H, KV, D, layers = MODELS[case["model"]]
    if kind == "rope":
        M, rot = case["M"], case["rot"]
        parents = _parents(g, M, M > 256)
        depth = _ancestors(parents).sum(1) - 1 if M <= 256 else torch.arange(M, device="cuda")
        last = case["pos"] + M
        angle = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * \
            THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        d = {"table": torch.cat([angle.cos(), angle.sin()], 1).float(), "pos": (case["pos"] + depth).int(),
             "q_norm": 1 + _normal(g, D, scale=0.1), "k_norm": 1 + _normal(g, D, scale=0.1)}
        if case["fused"]:
            d["qkv"] = _normal(g, M, (H + 2 * KV) * D)
        else:
            d.update(q=_normal(g, M, H * D), k=_normal(g, M, KV * D), v=_normal(g, M, KV * D))
        return d
    if kind == "tree":
        M, T, t = case["M"], case["past"] + case["M"], _TYPES[case["cache"]]
        return {"q": _normal(g, M, H * D, scale=2.0), "k": _normal(g, T, KV * D, dtype=t), "v": _normal(g, T, KV * D, dtype=t),
                "mask": _words(_ancestors(_parents(g, M, case["chain"])))}
    n, rows, t = case["n"], case["rows"], _TYPES[case["cache"]]
    if not rows:
        return {"cache": _normal(g, 2 * layers, n + 48, KV * D, dtype=t), "to": torch.zeros(2 * layers, n + 48, KV * D, dtype=t, device="cuda")}
    # An accepted path, ascending. What it takes lies where nothing is put, or stays, so that a second pass changes nothing.
    first = int(torch.randint(n, (1,), generator=g, device="cuda"))
    later = n + torch.randperm(rows - n, generator=g, device="cuda")[:n - first].sort().values
    path = torch.cat([torch.arange(n - later.numel(), device="cuda"), later]).int()
    return {"cache": _normal(g, 2 * layers, case["past"] + rows, KV * D, dtype=t), "path": path}


# ------------------------------------------------------------------ the library's side

_context = None


def _library():
    """The module and the one context (device, stream) that a program keeps."""
    global _context
    from webllm_amd import qlinear as ql
    if _context is None:
        _context = ql.Context(0)
    return ql, _context


class _Bytes:
    """Memory of an arena, which lives as long as a tensor over it."""

    def __init__(self, arena, off, shape, kind):
        self.arena = arena
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind, "version": 3,
                                         "data": (arena.device_ptr + off, False)}


_KINDS = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4", torch.int64: "<i8"}


class _Arena:
    """Tensors laid out in one device arena."""

    def __init__(self, ql, ctx, **tensors):
        lay = ql.ArenaLayout()
        self.off = {n: lay.take(max(16, t.numel() * t.element_size())) for n, t in tensors.items()}
        self.arena = ctx.arena(lay.used)
        for n, t in tensors.items():
            if t.numel():
                self.view(n, t.shape, t.dtype).copy_(t)

    def view(self, name, shape, dtype=torch.float32):
        return torch.as_tensor(_Bytes(self.arena, self.off[name], shape, _KINDS[dtype]), device="cuda")


class _Handles:
    pass


def _place(case, d):
    """A program's handles: call() is the call, outputs the arena memory that it fills."""
    ql, ctx = _library()
    s, kind = _Handles(), case["kind"]
    like = torch.empty
    if kind == "logprobs":
        M, V, T, top = case["M"], case["V"], case["T"], case["top"]
        f = {"device": "cuda"}
        a = _Arena(ql, ctx, logits=d["logits"], tokens=d["tokens"], lp=like(M, T, **f), ent=like(M, **f),
                   ids=like(M, top, dtype=torch.int32, **f), tlp=like(M, top, **f))
        o = a.off
        s.keep, args = a, (a.arena, o["logits"], V, M, V, o["tokens"], T, top, o["lp"], o["ent"], o["ids"], o["tlp"])
        s.call = lambda: ctx.token_logprobs(*args)
        s.outputs = {"entropy": a.view("ent", (M,))}
        if T:
            s.outputs["logprobs"] = a.view("lp", (M, T))
        if top:
            s.outputs.update(ids=a.view("ids", (M, top), torch.int32), top=a.view("tlp", (M, top)))
        return s
    H, KV, D, layers = MODELS[case["model"]]
    kind_of = ql.DTYPE_F16 if case["cache"] == "f16" else ql.DTYPE_F32
    t, size = _TYPES[case["cache"]], _BYTES[case["cache"]]
    if kind == "rope":
        M = case["M"]
        w = _Arena(ql, ctx, table=d["table"], q_norm=d["q_norm"], k_norm=d["k_norm"])
        inputs = {n: d[n] for n in ("qkv", "q", "k", "v") if n in d}
        a = _Arena(ql, ctx, pos=d["pos"], out=like(M, H * D, device="cuda"), **inputs)
        c = _Arena(ql, ctx, k=like(M, KV * D, dtype=t, device="cuda"), v=like(M, KV * D, dtype=t, device="cuda"))
        stride = (H + 2 * KV) * D if case["fused"] else 0
        qkv = [a.off["qkv"] + 4 * D * n for n in (0, H, H + KV)] if case["fused"] else [a.off[n] for n in "qkv"]
        rope = ql.make_rope(w.off["table"], d["table"].shape[0], H, KV, D, rot_dim=case["rot"], interleaved=case["interleaved"],
                            q_norm_off=w.off["q_norm"] if case["norm"] else None, k_norm_off=w.off["k_norm"] if case["norm"] else None,
                            norm_eps=EPS, q_stride=stride, k_stride=stride, v_stride=stride, cache_dtype=kind_of)
        s.keep, args = (w, a, c), (rope, w.arena, a.arena, *qkv, a.off["pos"], M, a.off["out"], c.arena, c.off["k"], c.off["v"], M, 0)
        s.call = lambda: ctx.qk_norm_rope(*args)
        s.outputs = [a.view("out", (M, H, D)), c.view("k", (M, KV, D), t), c.view("v", (M, KV, D), t)]
        return s
    if kind == "tree":
        M, past = case["M"], case["past"]
        a = _Arena(ql, ctx, q=d["q"], mask=d["mask"], out=like(M, H * D, device="cuda"))
        c = _Arena(ql, ctx, k=d["k"], v=d["v"])
        s.keep, args = (a, c), (a.arena, a.off["q"], c.arena, c.off["k"], c.off["v"], kind_of, past + M, M, H, KV, D, past, a.off["mask"],
                                a.off["out"])
        s.call = lambda: ctx.attention_tree(*args)
        s.outputs = [a.view("out", (M, H, D))]
        return s
    c = _Arena(ql, ctx, cache=d["cache"])
    T, row = d["cache"].shape[1], KV * D * size
    offs = ql.offsets([c.off["cache"] + i * T * row for i in range(2 * layers)])
    if "path" in d:
        a = _Arena(ql, ctx, path=d["path"])
        args = (c.arena, offs, T, c.arena, offs, T, row, case["past"], case["past"], case["n"], a.arena, a.off["path"])
        s.keep, s.outputs = (a, c), [c.view("cache", d["cache"].shape, t)[:, case["past"]:]]
    else:
        to = _Arena(ql, ctx, to=d["to"])
        args = (to.arena, ql.offsets([to.off["to"] + i * T * row for i in range(2 * layers)]), T, c.arena, offs, T, row, 0, 0, case["n"])
        s.keep, s.outputs = (c, to), [to.view("to", d["to"].shape, t)]
    s.call = lambda: ctx.kv_move(*args)
    return s


# ------------------------------------------------------------------ the formulas in torch

def _seen(mask, M):
    """[M, M] of a mask's words."""
    return ((mask[:, :, None] >> torch.arange(64, device="cuda")) & 1).reshape(M, -1)[:, :M].bool()


def _heads(case, d):
    H, KV, D, _ = MODELS[case["model"]]
    q, k, v = d["qkv"].split([H * D, KV * D, KV * D], 1) if case["fused"] else (d["q"], d["k"], d["v"])
    M = case["M"]
    return q.reshape(M, H, D), k.reshape(M, KV, D), v.reshape(M, KV, D)


def _rotate(case, d, x, norm):
    """Heads of x normed and their first `rot` values turned by their row's angles."""
    if case["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    rot = case["rot"]
    c, s = (t[:, None, :] for t in d["table"][d["pos"].long()].chunk(2, 1))
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def _plain(case, d):
    kind = case["kind"]
    if kind == "rope":
        q, k, v = _heads(case, d)
        t = _TYPES[case["cache"]]
        return [_rotate(case, d, q, d["q_norm"]), _rotate(case, d, k, d["k_norm"]).to(t), v.to(t)]
    if kind == "tree":
        H, KV, D, _ = MODELS[case["model"]]
        M, T, G = case["M"], d["k"].shape[0], H // KV
        q = d["q"].reshape(M, KV, G, D).permute(1, 0, 2, 3).reshape(KV, M * G, D)
        k = d["k"].float().reshape(T, KV, D).permute(1, 2, 0).contiguous()
        v = d["v"].float().reshape(T, KV, D).permute(1, 0, 2).contiguous()
        seen = torch.cat([torch.ones(M, case["past"], dtype=torch.bool, device="cuda"), _seen(d["mask"], M)], 1)
        score = torch.bmm(q, k).reshape(KV, M, G, T) * (1 / math.sqrt(D))
        score = score.masked_fill(~seen[None, :, None, :], -math.inf)
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - torch.where(top == -math.inf, 0.0, top)).reshape(KV, M * G, T)
        total = p.sum(-1, keepdim=True)
        out = torch.where(total > 0, torch.bmm(p, v) / total, 0.0)
        return [out.reshape(KV, M, G, D).permute(1, 0, 2, 3).reshape(M, H, D)]
    if kind == "logprobs":
        x, tokens, V, top = d["logits"], d["tokens"].long(), case["V"], case["top"]
        most = x.amax(1, keepdim=True)
        most = torch.where(most == -math.inf, 0.0, most)
        e = torch.exp(x - most)
        total = e.sum(1, keepdim=True)
        none = total == 0
        log = torch.log(total)
        out = {"entropy": torch.where(none, 0.0, log - torch.where(e > 0, e * (x - most), 0.0).sum(1, keepdim=True) / total)[:, 0]}
        if case["T"]:
            there = (tokens >= 0) & (tokens < V)
            lp = torch.where(none, -math.inf, x.gather(1, tokens.clamp(0, V - 1)) - most - log)
            out["logprobs"] = torch.where(there, lp, 0.0)
        if top:
            n = min(top, V)
            bits = (x + 0.0).view(torch.int32)
            key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * 2**32 + (2**32 - 1 - torch.arange(V, device="cuda"))
            ids = 2**32 - 1 - (key.topk(n, dim=1).values & (2**32 - 1))
            lp = torch.where(none, -math.inf, x.gather(1, ids) - most - log)
            out["ids"] = torch.nn.functional.pad(ids, (0, top - n), value=-1).int()
            out["top"] = torch.nn.functional.pad(lp, (0, top - n), value=-math.inf)
        return out
    if "path" in d:
        past = case["past"]
        d["cache"][:, past:past + case["n"]] = d["cache"][:, past + d["path"].long()]
        return [d["cache"][:, past:]]
    d["to"][:, :case["n"]] = d["cache"][:, :case["n"]]
    return [d["to"]]


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        s = _place(case, d)
    else:
        s = (case, d)
    torch.cuda.synchronize()
    return s


def run(state):
    if own:
        state.call()
        return state.outputs
    return _plain(*state)


# ------------------------------------------------------------------ what a call cannot do without

def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        M, V, T, top = case["M"], case["V"], case["T"], case["top"]
        return {"bytes": M * (4 * V + 8 * T + 8 * top + 4), "flops": 6 * M * V}
    H, KV, D, layers = MODELS[case["model"]]
    size, M = _BYTES[case["cache"]], case.get("M", 0)
    if kind == "rope":
        return {"bytes": M * ((H + 2 * KV) * D * 4 + H * D * 4 + 2 * KV * D * size + 4 * case["rot"] + 4) + (8 * D if case["norm"] else 0),
                "flops": M * (H + KV) * (3 * case["rot"] + (4 * D if case["norm"] else 0))}
    if kind == "tree":      # a token sees the context, itself and, in a chain, all before it
        past = case["past"]
        return {"bytes": 2 * (past + M) * KV * D * size + 8 * M * H * D + 8 * M * (-(-M // 64)),
                "flops": 4 * H * D * M * (past + ((M + 1) // 2 if case["chain"] else 1))}
    return {"bytes": 2 * 2 * layers * case["n"] * KV * D * size + (4 * case["n"] if case["rows"] else 0), "flops": 0}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_rope(case, d):
    H, KV, D, _ = MODELS[case["model"]]
    M, rot = case["M"], case["rot"]
    if case["fused"]:
        x = d["qkv"].double().view(M, H + 2 * KV, D)
    else:
        x = torch.cat([d[n].double().view(M, -1, D) for n in ("q", "k", "v")], 1)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), d["pos"].double()[:, None] * torch.exp(-2 * i / rot * math.log(THETA)))
    out = []
    for h, w in ((q, d["q_norm"]), (k, d["k_norm"])):
        if case["norm"]:
            h = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        if case["interleaved"]:
            z = torch.complex(h[..., 0:rot:2].contiguous(), h[..., 1:rot:2].contiguous()) * turn[:, None]
            r = torch.stack([z.real, z.imag], -1).flatten(-2)
        else:
            z = torch.complex(h[..., :rot // 2].contiguous(), h[..., rot // 2:rot].contiguous()) * turn[:, None]
            r = torch.cat([z.real, z.imag], -1)
        out.append(torch.cat([r, h[..., rot:]], -1))
    return out + [v]


def _exact_tree(case, d):
    H, KV, D, _ = MODELS[case["model"]]
    M, past, out = case["M"], case["past"], []
    at = torch.arange(M, device="cuda")
    tail = (d["mask"][:, at // 64] >> (at % 64)) & 1
    hide = torch.nn.functional.pad(tail == 0, (past, 0))
    for h in range(H):
        kv = slice(h // (H // KV) * D, (h // (H // KV) + 1) * D)
        s = d["q"][:, h * D:(h + 1) * D].double() @ d["k"][:, kv].double().T.contiguous() / math.sqrt(D)
        s[hide] = -math.inf
        w = torch.softmax(s, 1)
        out.append(torch.nan_to_num(w) @ d["v"][:, kv].double())
    return [torch.stack(out, 1)]


def _exact_logprobs(case, d):
    M, V, T, top = case["M"], case["V"], case["T"], case["top"]
    out = {"entropy": [], "logprobs": [], "ids": [], "top": []}
    for m in range(M):
        x = d["logits"][m].double()
        lp = torch.log_softmax(x, 0) if bool((x > -math.inf).any()) else x
        out["entropy"].append(-(torch.exp(lp) * lp)[lp > -math.inf].sum())
        if T:
            t = d["tokens"][m].long()
            out["logprobs"].append(torch.where((t >= 0) & (t < V), lp[t.clamp(0, V - 1)], 0.0))
        if top:
            order = torch.sort(x, descending=True, stable=True).indices[:top]
            more = top - order.numel()
            out["ids"].append(torch.cat([order, order.new_full((more,), -1)]))
            out["top"].append(torch.cat([lp[order], lp.new_full((more,), -math.inf)]))
    out = {n: torch.stack(v) for n, v in out.items() if v}
    if top:
        out["ids"] = out["ids"].int()
    return out


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    if kind == "rope":
        return _exact_rope(case, d)
    if kind == "tree":
        return _exact_tree(case, d)
    if kind == "logprobs":
        return _exact_logprobs(case, d)
    cache, n, past = d["cache"].double(), case["n"], case["past"]
    if "path" not in d:
        return [torch.cat([cache[:, :n], d["to"][:, n:].double()], 1)]
    from_rows = past + torch.cat([d["path"].long(), torch.arange(n, case["rows"], device="cuda")])
    return [cache.index_select(1, from_rows)]
