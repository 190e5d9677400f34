"""The operators of a pass over many requests at once as cases that can be timed and checked: rotating a batch's queries and keys
and appending keys and values to a paged cache, attention of the batch's rows over that cache, and the low-rank adapters of the
batch's requests beside a shared projection.

Each case is one call. Where `own` is false, `run` is the operator's formula in elementary torch operations; where it is
true, the call of webllm_amd.qlinear that computes it, on inputs that lie in the library's arenas. `exact` is the same in
64-bit arithmetic.

A batch has sequences of some rows each: one row of a request that decodes, many of a prompt or of a piece of one. Its rows lie
one sequence behind the other. Row i of a sequence that has n rows in the batch and L tokens with them is token L - n + i. Token t of
a sequence lies in the page that the sequence's list names at t / page. A cache of 8 bits holds e4m3 values and, for every 16 tokens of a
page and every kv head, a power of two that they are multiplied by: the smallest under which the largest is at most 448, or a larger one
that the 16 tokens had before.
"""
import math
import random

import torch

own = False

# (heads, kv heads, head dim, width, mlp width) of the two model shapes that the benchmark and the tests use.
MODELS = {"05b": (14, 2, 64, 896, 4864), "7b": (28, 4, 128, 3584, 18944)}
THETA = 1e6
EPS = 1e-6
LEAST = -120                # exponent of the smallest power of two of an 8-bit cache


def listed():
    return [
        # Four chats of the small model, one token each: rotation, append, launch latency.
        {"name": "append_05b_s4", "kind": "append", "model": "05b", "dec": 4, "T": 500, "prompts": 0, "rows": 0, "past": 0, "pad": 0,
         "page": 64, "cache": "f16", "q": "f32", "norm": False, "rot": 64, "interleaved": False, "fused": False},
        # A server's decoding batch: 64 requests, an 8-bit cache, heads normed, rows of one fused projection.
        {"name": "append_7b_s64_f8", "kind": "append", "model": "7b", "dec": 64, "T": 1500, "prompts": 0, "rows": 0, "past": 0, "pad": 0,
         "page": 64, "cache": "f8", "q": "f32", "norm": True, "rot": 128, "interleaved": False, "fused": True},
        # Five prompts of 4096 tokens together into an 8-bit cache: a stream through memory.
        {"name": "append_7b_prompts_f8", "kind": "append", "model": "7b", "dec": 0, "T": 0, "prompts": 5, "rows": 4096, "past": 0, "pad": 0,
         "page": 128, "cache": "f8", "q": "f16", "norm": False, "rot": 128, "interleaved": False, "fused": False},
        # Four chats of some hundred tokens: latency.
        {"name": "attn_05b_s4_t300", "kind": "attn", "model": "05b", "dec": 4, "T": 300, "prompts": 0, "rows": 0, "past": 0, "pad": 0,
         "page": 64, "cache": "f16", "q": "f32"},
        # A server's decoding batch: 64 requests of 800 to 8000 tokens, an 8-bit cache: memory-bound, ragged.
        {"name": "attn_7b_s64_t8000_f8", "kind": "attn", "model": "7b", "dec": 64, "T": 8000, "prompts": 0, "rows": 0, "past": 0, "pad": 0,
         "page": 64, "cache": "f8", "q": "f32"},
        # One request over a long document: its keys over the whole chip.
        {"name": "attn_7b_s1_t60000", "kind": "attn", "model": "7b", "dec": 1, "T": 60000, "prompts": 0, "rows": 0, "past": 0, "pad": 0,
         "page": 256, "cache": "f16", "q": "f32"},
        # Five whole prompts of 9000 tokens in all, packed, fp16 rows: matrix-core bound. The largest.
        {"name": "attn_7b_prompts", "kind": "attn", "model": "7b", "dec": 0, "T": 0, "prompts": 5, "rows": 9000, "past": 0, "pad": 0,
         "page": 64, "cache": "f16", "q": "f16"},
        # Pieces of two long prompts in a batch that decodes, with rows of padding behind it.
        {"name": "attn_7b_mixed_f8", "kind": "attn", "model": "7b", "dec": 24, "T": 4000, "prompts": 2, "rows": 700, "past": 3500, "pad": 44,
         "page": 128, "cache": "f8", "q": "f16"},
        # Eight prompts of the small model, fp32 rows.
        {"name": "attn_05b_prompts", "kind": "attn", "model": "05b", "dec": 0, "T": 0, "prompts": 8, "rows": 2500, "past": 0, "pad": 0,
         "page": 64, "cache": "f16", "q": "f32"},
        # Four chats, three adapters, one row without: q, k and v of the small model.
        {"name": "lora_05b_m4", "kind": "lora", "model": "05b", "to": "qkv", "M": 4, "n": 3, "rank": 8, "x": "f32", "runs": False},
        # A decoding batch of 64 requests with 24 adapters between them.
        {"name": "lora_7b_m64", "kind": "lora", "model": "7b", "to": "qkv", "M": 64, "n": 24, "rank": 16, "x": "f32", "runs": False},
        # Prompts of 4096 tokens with four adapters, fp16 rows: a stream through memory.
        {"name": "lora_7b_prompts", "kind": "lora", "model": "7b", "to": "qkv", "M": 4096, "n": 4, "rank": 64, "x": "f16", "runs": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "attn", "lora", "lora"])
    model = rng.choice(["05b", "7b"])
    if kind == "lora":
        M = _log(rng, 1, 4096)
        to = rng.choice(["qkv", "qkv", "o", "up", "down"])
        while to in ("up", "down") and M > 512:
            M //= 2
        return {"kind": kind, "model": model, "to": to, "M": M, "n": _log(rng, 1, 40), "rank": rng.choice([8, 16, 16, 24, 32, 64]),
                "x": rng.choice(["f32", "f16"]), "runs": M > 64 or rng.random() < 0.3}
    D = MODELS[model][2]
    mix = rng.choice(["dec", "dec", "prompts", "both"])
    c = {"kind": kind, "model": model, "dec": 0, "T": 0, "prompts": 0, "rows": 0, "past": 0, "pad": rng.choice([0, 0, rng.randint(1, 100)]),
         "page": rng.choice([64, 128, 256]), "cache": rng.choice(["f16", "f8"]), "q": rng.choice(["f32", "f16"])}
    if kind == "append":
        c.update(norm=rng.random() < 0.5, rot=rng.choice([D, D, D // 2]), interleaved=rng.random() < 0.3, fused=rng.random() < 0.4)
    if mix != "prompts":
        c["dec"] = _log(rng, 1, 96)
        c["T"] = _log(rng, 16, 2000 if kind == "append" else 40000)
        while c["dec"] * c["T"] > 64 * 5000:
            c["T"] //= 2
    if mix != "dec":
        c["prompts"] = rng.randint(1, 6)
        c["rows"] = max(c["prompts"] * 2, _log(rng, 8, 4000))
        c["past"] = rng.choice([0, _log(rng, 16, 500 if kind == "append" else 12000)])
        while c["rows"] * (c["past"] + c["rows"] / c["prompts"]) > 7e6:
            c["rows"], c["past"] = max(c["prompts"] * 2, c["rows"] // 2), c["past"] // 2
    return c


def _sequences(case):
    """(rows in the batch, tokens with them) of each sequence, in the batch's order: a matter of the case alone."""
    rng = random.Random("%(dec)d %(T)d %(prompts)d %(rows)d %(past)d" % case)
    seqs = [(1, case["T"] if i == 0 else max(1, int(case["T"] * rng.uniform(0.1, 1)))) for i in range(case["dec"])]
    share = [rng.uniform(0.4, 1.6) for _ in range(case["prompts"])]
    for i, s in enumerate(share):
        n = max(1, int(case["rows"] * s / sum(share)))
        seqs.append((n, n + (case["past"] if i == 0 else int(case["past"] * rng.uniform(0.3, 1)))))
    rng.shuffle(seqs)
    return seqs


def _targets(case):
    """(inputs, outputs) of the projections that the adapters stand beside."""
    H, KV, D, C, I = MODELS[case["model"]]
    return {"qkv": [(C, H * D), (C, KV * D), (C, KV * D)], "o": [(H * D, C)], "up": [(C, I), (C, I)], "down": [(I, C)]}[case["to"]]


# ------------------------------------------------------------------ inputs, from the seed alone

_TYPES = {"f32": torch.float32, "f16": torch.float16, "f8": torch.float8_e4m3fn}
_BYTES = {"f32": 4, "f16": 2, "f8": 1}


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _power(top):
    """The smallest power of two p with top <= 448 p, no smaller than 2^LEAST."""
    m, e = torch.frexp(top / 448)
    e = torch.where(m == 0.5, e - 1, e)                  # top / 448 is one itself
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, LEAST).clamp(min=LEAST))


def _pages(case, g):
    """row_start [S + 1], kv_len [S], pages [S, most] (int32), and how many pages the cache has: every sequence has its own."""
    seqs, page = _sequences(case), case["page"]
    need = [-(-L // page) for _, L in seqs]
    total, most = sum(need) + 3, max(need)
    free, table, at = torch.randperm(total, generator=g, device="cuda").int(), [], 0
    for k in need:
        table.append(torch.nn.functional.pad(free[at:at + k], (0, most - k), value=-1))
        at += k
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    d = {"row_start": torch.tensor(starts, dtype=torch.int32, device="cuda"), "kv_len": torch.tensor([L for _, L in seqs], dtype=torch.int32, device="cuda"),
         "pages": torch.stack(table)}
    return d, total, starts[-1] + case["pad"]


def _inputs(case, seed):
    g, kind = torch.Generator(device="cuda").manual_seed(int(seed)), case["kind"]
    if kind == "lora":
        M, n, r = case["M"], case["n"], case["rank"]
        if case["runs"]:                                                             # requests' rows lie together
            ids = torch.sort(torch.randint(0, n + 1, (M,), generator=g, device="cuda")).values - 1
        else:
            ids = torch.randint(-1, n, (M,), generator=g, device="cuda")
        d = {"ids": ids.int(), "x": [], "a": [], "b": [], "base": [], "scale": []}
        for k, (K, N) in enumerate(_targets(case)):
            # q, k and v (gate and up) read one input
            d["x"].append(d["x"][0] if k else _normal(g, M, K, dtype=_TYPES[case["x"]]))
            d["a"].append(_normal(g, n, r, K, scale=K ** -0.5, dtype=torch.float16))
            d["b"].append(_normal(g, n, N, r, scale=r ** -0.5, dtype=torch.float16))
            d["base"].append(_normal(g, M, N))
            d["scale"].append(0.5 + torch.rand(n, generator=g, device="cuda"))
        return d
    H, KV, D, _, _ = MODELS[case["model"]]
    d, total, M = _pages(case, g)
    page, t = case["page"], _TYPES[case["cache"]]
    for n in ("k_cache", "v_cache"):
        x = _normal(g, total, page, KV, D)
        if case["cache"] == "f8":
            p = _power(x.view(total, page // 16, 16, KV, D).abs().amax((2, 4)))      # [pages, page / 16, kv heads]
            d[n[0] + "_scale"] = p
            x = x / p.repeat_interleave(16, 1)[..., None]
        d[n] = x.to(t)
    if kind == "attn":
        d["q"] = _normal(g, M, H, D, scale=2.0, dtype=_TYPES[case["q"]])
        return d
    rot, last = case["rot"], max(L for _, L in _sequences(case))
    angle = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * \
        THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    d.update(table=torch.cat([angle.cos(), angle.sin()], 1).float(), q_norm=1 + _normal(g, D, scale=0.1), k_norm=1 + _normal(g, D, scale=0.1))
    if case["fused"]:
        d["qkv"] = _normal(g, M, (H + 2 * KV) * D)
    else:
        d.update(q=_normal(g, M, H * D), k=_normal(g, M, KV * D), v=_normal(g, M, KV * D))
    return d


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


_KINDS = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4", torch.float8_e4m3fn: "|u1"}


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
        x = torch.as_tensor(_Bytes(self.arena, self.off[name], shape, _KINDS[dtype]), device="cuda")
        return x.view(dtype) if dtype == torch.float8_e4m3fn else x


class _Handles:
    pass


def _laid(case, d):
    """The caches' values in the order that the library keeps them. A kv head's 16 tokens of K are one block, 16 bytes of a token
    behind the other tokens' of the same columns; V's tokens come in fours, those of 32 (16 bits) or 64 (8 bits) tokens together,
    16 bytes of a column behind the next column's, 16 columns together."""
    total, page, KV, D = d["k_cache"].shape
    size = _BYTES[case["cache"]]
    u, many = 16 // size, 64 // size
    raw = {n: d[n].view(torch.uint8) if size == 1 else d[n] for n in ("k_cache", "v_cache")}
    k = raw["k_cache"].view(total, page // 16, 16, KV, D // u, u).permute(0, 3, 1, 4, 2, 5)
    v = raw["v_cache"].view(total, page // many, many // 16, 4, 4, KV, D // 16, 16).permute(0, 5, 1, 6, 3, 7, 2, 4)
    t = _TYPES[case["cache"]]
    out = {"k": k.contiguous().view(t), "v": v.contiguous().view(t)}
    if size == 1:
        out.update({n: d[n].transpose(1, 2).contiguous() for n in ("k_scale", "v_scale")})
    return out


def _shown(c, case, shapes):
    """Views of the library's caches with the tokens in order, as _plain returns them."""
    t = _TYPES[case["cache"]]
    out = {"k": c.view("k", shapes["k"], t).permute(0, 2, 4, 1, 3, 5), "v": c.view("v", shapes["v"], t).permute(0, 2, 6, 4, 7, 1, 3, 5)}
    if case["cache"] == "f8":
        out.update({n: c.view(n, shapes[n]).transpose(1, 2) for n in ("k_scale", "v_scale")})
    return out


def _place(case, d):
    """A program's handles: call() is the call, outputs the arena memory that it fills."""
    ql, ctx = _library()
    s, kind = _Handles(), case["kind"]
    kind_of = {"f32": ql.DTYPE_F32, "f16": ql.DTYPE_F16}
    if kind == "lora":
        count, targets = len(d["a"]), _targets(case)
        w = _Arena(ql, ctx, **{n + str(i): d[n][i] for i in range(count) for n in ("a", "b", "scale")})
        a = _Arena(ql, ctx, ids=d["ids"], x=d["x"][0], **{"base%d" % i: d["base"][i] for i in range(count)},
                   **{"y%d" % i: torch.empty_like(d["base"][i]) for i in range(count)})
        descs = ql.lora_descs([ql.make_lora(w.off["a%d" % i], w.off["b%d" % i], K, N, case["rank"], case["n"], scale_off=w.off["scale%d" % i])
                               for i, (K, N) in enumerate(targets)])
        xs, bases, ys = (ql.offsets([a.off[n] for n in names]) for names in
                         (["x"] * count, ["base%d" % i for i in range(count)], ["y%d" % i for i in range(count)]))
        s.keep, args = (w, a), (descs, w.arena, a.arena, a.off["ids"], xs, kind_of[case["x"]], case["M"], bases, ys)
        s.call = lambda: ctx.lora_add(*args)
        s.outputs = [a.view("y%d" % i, d["base"][i].shape) for i in range(count)]
        return s
    H, KV, D, _, _ = MODELS[case["model"]]
    seqs = _sequences(case)
    laid, M = _laid(case, d), sum(n for n, _ in seqs) + case["pad"]
    shapes = {n: x.shape for n, x in laid.items()}
    c = _Arena(ql, ctx, **laid)
    tables = {n: d[n] for n in ("row_start", "kv_len", "pages")}
    out = torch.zeros(M, H, D, dtype=_TYPES[case["q"]], device="cuda")
    inputs = {n: d[n] for n in ("qkv", "q", "k", "v") if n in d}
    a = _Arena(ql, ctx, out=out, **inputs, **tables)
    paged = ql.make_paged(c.off["k"], c.off["v"], laid["k"].shape[0], case["page"], KV, D,
                          cache_dtype=ql.DTYPE_F8 if case["cache"] == "f8" else ql.DTYPE_F16,
                          k_scale_off=c.off.get("k_scale"), v_scale_off=c.off.get("v_scale"))
    batch = ql.make_batch(a.off["row_start"], a.off["kv_len"], a.off["pages"], len(seqs), d["pages"].shape[1],
                          max_rows=max(n for n, _ in seqs), max_len=max(L for _, L in seqs))
    s.outputs = {"out": a.view("out", (M, H, D), _TYPES[case["q"]])}
    if kind == "attn":
        args = (a.arena, a.off["q"], kind_of[case["q"]], c.arena, paged, batch, M, H, a.off["out"])
        s.keep, s.call = (a, c), lambda: ctx.paged_attention(*args)
        return s
    w = _Arena(ql, ctx, table=d["table"], q_norm=d["q_norm"], k_norm=d["k_norm"])
    stride = (H + 2 * KV) * D if case["fused"] else 0
    qkv = [a.off["qkv"] + 4 * D * n for n in (0, H, H + KV)] if case["fused"] else [a.off[n] for n in "qkv"]
    rope = ql.make_rope(w.off["table"], d["table"].shape[0], H, KV, D, rot_dim=case["rot"], interleaved=case["interleaved"],
                        q_norm_off=w.off["q_norm"] if case["norm"] else None, k_norm_off=w.off["k_norm"] if case["norm"] else None,
                        norm_eps=EPS, q_stride=stride, k_stride=stride, v_stride=stride, cache_dtype=paged.cache_dtype)
    args = (rope, w.arena, a.arena, *qkv, batch, M, a.off["out"], kind_of[case["q"]], c.arena, paged)
    s.keep, s.call = (a, c, w), lambda: ctx.paged_append(*args)
    s.outputs.update(_shown(c, case, shapes))
    return s


# ------------------------------------------------------------------ the formulas in torch

def _rows(case, d, M):
    """Of each row of the batch: its sequence, its token, and whether it is one and no padding."""
    m = torch.arange(M, device="cuda")
    ends = d["row_start"][1:].long()
    there = m < ends[-1]
    seq = torch.bucketize(m, ends, right=True).clamp(max=ends.numel() - 1)
    return seq, torch.where(there, d["kv_len"].long()[seq] - ends[seq] + m, 0), there


def _rotate(case, d, x, norm, pos):
    """Heads of x normed and their first `rot` values turned by their row's angles."""
    if case["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    rot = case["rot"]
    c, s = (t[:, None, :] for t in d["table"][pos].chunk(2, 1))
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def _heads(case, d, M):
    H, KV, D, _, _ = MODELS[case["model"]]
    q, k, v = d["qkv"].split([H * D, KV * D, KV * D], 1) if case["fused"] else (d["q"], d["k"], d["v"])
    return q.reshape(M, H, D), k.reshape(M, KV, D), v.reshape(M, KV, D)


def _put(cache, scale, x, at, start):
    """Rows x at tokens `at` of a cache of 8 bits; start: the first of the row's 16 tokens that the batch brings."""
    total, page, KV, D = cache.shape
    flat, scales = cache.view(-1, 16, KV, D), scale.view(-1, KV)
    block, slot = at // 16, at % 16
    top = torch.zeros(flat.shape[0], KV, device="cuda").index_reduce_(0, block, x.abs().amax(2), "amax")[block]
    before = scales[block]
    now = torch.where((start > 0)[:, None], torch.maximum(before, _power(top)), _power(top))       # [rows, kv heads]
    keep = torch.arange(16, device="cuda") < start[:, None]
    moved = (flat[block].float() * (before / now)[:, None, :, None]).to(cache.dtype)
    raw = flat.view(torch.uint8)
    raw[block] = torch.where(keep[:, :, None, None], moved.view(torch.uint8), raw[block])
    scales[block] = now
    raw[block, slot] = (x / now[..., None]).to(cache.dtype).view(torch.uint8)


def _cached(d, name, seq, tokens):
    """[sequences, tokens, kv heads, D] of a cache in fp32."""
    cache = d[name + "_cache"]
    page = cache.shape[1]
    row = d["pages"][seq].long().gather(1, (tokens // page).expand(len(seq), -1)).clamp(min=0) * page + tokens % page
    x = cache.view(-1, *cache.shape[2:])
    x = (x.view(torch.uint8)[row].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[row]).float()
    return x * d[name + "_scale"].view(-1, cache.shape[2])[row // 16][..., None] if name + "_scale" in d else x


def _attend(case, d, out, seq, n, most):
    """Sequences `seq` (a list) of at most n rows and `most` tokens."""
    H, KV, D, _, _ = MODELS[case["model"]]
    G, S = H // KV, len(seq)
    seq = torch.tensor(seq, device="cuda")
    first, rows, L = d["row_start"].long()[seq][:, None], d["row_start"].diff().long()[seq][:, None], d["kv_len"].long()[seq][:, None]
    i, t = torch.arange(n, device="cuda")[None], torch.arange(most, device="cuda")[None]
    there = t < L
    k, v = (torch.where(there[..., None, None], _cached(d, x, seq, t.clamp(max=case["page"] * d["pages"].shape[1] - 1)), 0.0) for x in "kv")
    q = d["q"][torch.minimum(first + i, first + rows - 1)].float().view(S, n, KV, G, D).permute(0, 2, 1, 3, 4).reshape(S * KV, n * G, D)
    score = torch.bmm(q, k.permute(0, 2, 3, 1).reshape(S * KV, D, most).contiguous()).view(S, KV, n, G, most) * (1 / math.sqrt(D))
    seen = t[:, None] <= (L - rows + i)[..., None]
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_().view(S * KV, n * G, most)
    o = torch.bmm(p, v.permute(0, 2, 1, 3).reshape(S * KV, most, D).contiguous()) / p.sum(-1, keepdim=True)
    used = (i < rows).reshape(-1)
    out[(first + i).reshape(-1)[used]] = o.view(S, KV, n, G, D).permute(0, 2, 1, 3, 4).reshape(S * n, H, D)[used].to(out.dtype)


def _plain(case, d):
    kind = case["kind"]
    if kind == "lora":
        out = []
        mine = (d["ids"][:, None] == torch.arange(case["n"], device="cuda"))[:, :, None]           # [M, n, 1]
        for x, a, b, base, scale in zip(d["x"], d["a"], d["b"], d["base"], d["scale"]):
            t = torch.mm(x.float(), a.float().flatten(0, 1).T).view(len(x), case["n"], case["rank"])
            t = torch.where(mine, t * scale[:, None], 0.0).flatten(1)
            out.append(base + torch.mm(t, b.float().permute(0, 2, 1).flatten(0, 1)))
        return out
    H, KV, D, _, _ = MODELS[case["model"]]
    seqs = _sequences(case)
    M = sum(n for n, _ in seqs) + case["pad"]
    out = torch.zeros(M, H, D, dtype=_TYPES[case["q"]], device="cuda")
    if kind == "attn":
        for one in (True, False):                                                    # requests of one row, and the others
            some = [s for s, (n, _) in enumerate(seqs) if (n == 1) == one]
            if some:
                _attend(case, d, out, some, max(seqs[s][0] for s in some), max(seqs[s][1] for s in some))
        return {"out": out}
    q, k, v = _heads(case, d, M)
    seq, pos, there = _rows(case, d, M)
    out[there] = _rotate(case, d, q, d["q_norm"], pos)[there].to(out.dtype)
    k = _rotate(case, d, k, d["k_norm"], pos)[there]
    seq, pos, page = seq[there], pos[there], case["page"]
    at = d["pages"].long()[seq, pos // page] * page + pos % page
    start = ((d["kv_len"] - d["row_start"].diff()).long()[seq] - pos // 16 * 16).clamp(min=0)
    for name, x in (("k", k), ("v", v[there])):
        if case["cache"] == "f8":
            _put(d[name + "_cache"], d[name + "_scale"], x, at, start)
        else:
            d[name + "_cache"].view(-1, KV, D)[at] = x.half()
    return {"out": out, **_in_order(case, d["k_cache"], d["v_cache"]), **{n: d[n] for n in ("k_scale", "v_scale") if n in d}}


def _in_order(case, k, v):
    """K and V of [pages, tokens, kv heads, D] in the dimensions in which the library's are shown."""
    total, page, KV, D = k.shape
    u, many = 16 // _BYTES[case["cache"]], 64 // _BYTES[case["cache"]]
    return {"k": k.view(total, page // 16, 16, KV, D // u, u), "v": v.view(total, page // many, many // 16, 4, 4, KV, D // 16, 16)}


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
    if kind == "lora":
        M, n, r, size = case["M"], case["n"], case["rank"], _BYTES[case["x"]]
        read, flops = 4 * M + size * M * _targets(case)[0][0], 0
        for K, N in _targets(case):
            read += 2 * min(n, M) * r * (K + N) + 8 * M * N
            flops += 2 * M * r * (K + N)
        return {"bytes": read, "flops": flops}
    H, KV, D, _, _ = MODELS[case["model"]]
    seqs, size, q = _sequences(case), _BYTES[case["cache"]], _BYTES[case["q"]]
    rows, pages = sum(n for n, _ in seqs), sum(-(-L // case["page"]) for _, L in seqs)
    row = 2 * KV * (D * size + (0.25 if size == 1 else 0))           # K and V of a token, and its share of the scales
    if kind == "append":
        return {"bytes": rows * ((H + 2 * KV) * D * 4 + H * D * q + row + 4 * case["rot"] + 4) + 8 * len(seqs) + (8 * D if case["norm"] else 0),
                "flops": rows * (H + KV) * (3 * case["rot"] + (4 * D if case["norm"] else 0))}
    return {"bytes": sum(L for _, L in seqs) * row + 2 * rows * H * D * q + 4 * pages + 8 * len(seqs),
            "flops": 4 * H * D * sum(n * (L - n) + n * (n + 1) // 2 for n, L in seqs)}


# ------------------------------------------------------------------ the same in 64 bits

def _values(d, name):
    """A cache's numbers, [tokens of all pages, kv heads, D]."""
    x = d[name + "_cache"].double()
    if name + "_scale" in d:
        x = x * d[name + "_scale"].double().repeat_interleave(16, 1)[..., None]
    return x.flatten(0, 1)


def _places(case, d, s, L):
    t = torch.arange(L, device="cuda")
    return d["pages"][s].long()[t // case["page"]] * case["page"] + t % case["page"]


def _exact_attn(case, d):
    H, KV, D, _, _ = MODELS[case["model"]]
    out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    k, v, row = _values(d, "k"), _values(d, "v"), 0
    for s, (n, L) in enumerate(_sequences(case)):
        at = _places(case, d, s, L)
        for h in range(H):
            kh, vh = k[at, h // (H // KV)], v[at, h // (H // KV)]
            for lo in range(0, n, 2048):
                hi = min(n, lo + 2048)
                x = d["q"][row + lo:row + hi, h].double() @ kh.T.contiguous() / math.sqrt(D)
                x += torch.full_like(x, -math.inf).triu(L - n + lo + 1)
                out[row + lo:row + hi, h] = torch.softmax(x, 1) @ vh
        row += n
    return {"out": out}


def _exact_append(case, d):
    H, KV, D, _, _ = MODELS[case["model"]]
    rot, seqs = case["rot"], _sequences(case)
    rows = sum(n for n, _ in seqs)
    if case["fused"]:
        x = d["qkv"][:rows].double().view(rows, H + 2 * KV, D)
    else:
        x = torch.cat([d[n][:rows].double().view(rows, -1, D) for n in ("q", "k", "v")], 1)
    pos = torch.cat([torch.arange(L - n, L, device="cuda", dtype=torch.float64) for n, L in seqs])
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[:, None] * torch.exp(-2 * i / rot * math.log(THETA)))[:, None]
    new = {"v": x[:, H + KV:]}
    for name, h, w in (("out", x[:, :H], d["q_norm"]), ("k", x[:, H:H + KV], d["k_norm"])):
        if case["norm"]:
            h = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        if case["interleaved"]:
            z = torch.complex(h[..., 0:rot:2].contiguous(), h[..., 1:rot:2].contiguous()) * turn
            r = torch.stack([z.real, z.imag], -1).flatten(-2)
        else:
            z = torch.complex(h[..., :rot // 2].contiguous(), h[..., rot // 2:rot].contiguous()) * turn
            r = torch.cat([z.real, z.imag], -1)
        new[name] = torch.cat([r, h[..., rot:]], -1)
    out = {"out": torch.nn.functional.pad(new["out"], (0, 0, 0, 0, 0, case["pad"]))}
    where = torch.cat([_places(case, d, s, L)[L - n:] for s, (n, L) in enumerate(seqs)])
    cache = {}
    for name in "kv":
        all_of = _values(d, name)
        if case["cache"] == "f8":
            # a group of 16 tokens keeps its power of two while what is new fits under it; a group that begins anew has the least
            power, row = d[name + "_scale"].double().clone(), 0
            groups = power.view(-1, KV)
            for s, (n, L) in enumerate(seqs):
                for t0 in range((L - n) // 16 * 16, L, 16):
                    a, b = max(t0, L - n), min(t0 + 16, L)
                    top = new[name][row + a - (L - n):row + b - (L - n)].abs().amax((0, 2))
                    least = torch.pow(2.0, torch.ceil(torch.log2(top / 448)).clamp(min=LEAST))
                    g = where[row + a - (L - n)] // 16
                    groups[g] = torch.maximum(groups[g], least) if a > t0 else least
                row += n
            # what stands beyond the sequences' ends has no meaning: its 8 bits stay
            old = d[name + "_cache"].double().view(-1, 16, KV, D)
            first = torch.full((old.shape[0],), 16, device="cuda")
            for s, (n, L) in enumerate(seqs):
                if L % 16:
                    first[_places(case, d, s, L)[-1] // 16] = L % 16
            beyond = torch.arange(16, device="cuda") >= first[:, None]
            all_of[where] = new[name]
            units = all_of.view(-1, 16, KV, D) / groups[:, None, :, None]
            cache[name] = torch.where(beyond[:, :, None, None], old, units).view(d[name + "_cache"].shape)
            out[name + "_scale"] = power
        else:
            all_of[where] = new[name]
            cache[name] = all_of.view(d[name + "_cache"].shape)
    return {**out, **_in_order(case, cache["k"], cache["v"])}


def _exact_lora(case, d):
    out = []
    for x, a, b, base, scale in zip(d["x"], d["a"], d["b"], d["base"], d["scale"]):
        y = base.double()
        for n in range(case["n"]):
            m = (d["ids"] == n).nonzero()[:, 0]
            y[m] += scale[n].double() * ((x[m].double() @ a[n].double().T.contiguous()) @ b[n].double().T.contiguous())
        out.append(y)
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "lora": _exact_lora}[case["kind"]](case, d)
