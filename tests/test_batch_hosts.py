"""Passes over many requests through the Python host (webllm_amd.gptq): sequences' pages on the CPU, with a context that records its calls in
place of the device's; and a model with adapters over several sequences, in the order a program has it, on the GPU."""
import numpy as np
import pytest

from tests.paged_ref import f8_decode, f8_encode, power
from tests.test_draft import CFG, Model, turned
from tests.test_draft_hosts import model_of, tensors
from tests.test_gpu_attn_tree import formula as attention
from webllm_amd import gptq
from webllm_amd import qlinear as ql


class Held:
    """An arena that keeps what is written."""

    def __init__(self, size):
        self.size, self.data = size, {}

    def write(self, off, a):
        self.data[off] = np.array(a)


class Context:
    def __init__(self):
        self.log = []

    def arena(self, n):
        return Held(n)

    def __getattr__(self, call):
        return lambda *args: self.log.append((call, args))


def cache_of(pages, page_size=64, dtype="f8"):
    ctx = Context()
    return ctx, gptq.PagedKvCache(ctx, CFG, pages, page_size, dtype), gptq.ActivationArena(ctx, 1 << 20)


def tables(batch):
    return [t.arena.data[t.offset] for t in batch.tables]


def test_pages_of_sequences():
    ctx, kv, pool = cache_of(8)
    a, b = kv.new_sequence(), kv.new_sequence()
    one = kv.batch(pool, [(a, 70), (b, 1)])
    start, lens, pages = tables(one)
    assert list(start) == [0, 70, 71] and list(lens) == [70, 1] and pages.shape == (2, 2) and pages[1, 1] == -1
    assert (one.M, one.rows, one.desc.n_seq, one.desc.max_pages, one.desc.max_rows, one.desc.max_len) == (71, 71, 2, 2, 70, 70)
    assert len({*pages[0], pages[1, 0]}) == 3 and kv.free_pages == 5 and kv.length(a) == 70
    two = kv.batch(pool, [(b, 63), (a, 0)], M=80)                               # fills its page exactly; other order; padding
    start, lens, pages2 = tables(two)
    assert list(start) == [0, 63, 63] and list(lens) == [64, 70] and (two.M, two.rows) == (80, 63) and kv.free_pages == 5
    assert pages2[0, 0] == pages[1, 0] and list(pages2[1]) == list(pages[0])
    kv.batch(pool, [(b, 1)])
    assert kv.free_pages == 4
    kv.free(a)
    assert kv.free_pages == 6
    with pytest.raises(KeyError):
        kv.length(a)
    kv.cut(b, 64)
    assert kv.free_pages == 7 and kv.length(b) == 64
    kv.cut(b, 0)
    assert kv.free_pages == 8
    assert not ctx.log


def test_batches_that_are_none():
    ctx, kv, pool = cache_of(3)
    a, b = kv.new_sequence(), kv.new_sequence()
    kv.batch(pool, [(a, 100)])
    for call in (lambda: kv.batch(pool, []), lambda: kv.batch(pool, [(a, 1), (a, 1)]), lambda: kv.batch(pool, [(a, -1)]), lambda: kv.batch(pool, [(a, 5)], M=4),
                 lambda: kv.batch(pool, [(a, 10), (b, 65)]), lambda: kv.cut(a, 101), lambda: kv.desc(CFG.n_layer)):
        with pytest.raises(ValueError):
            call()
    assert kv.length(a) == 100 and kv.length(b) == 0 and kv.free_pages == 1      # a refused batch takes nothing
    for kw in (dict(pages=0), dict(page_size=32), dict(dtype="f32")):
        with pytest.raises(ValueError):
            gptq.PagedKvCache(ctx, CFG, **{"pages": 4, **kw})


def test_pages_that_two_append_to():
    """Two sequences cut within a page that both hold: one copy, if nobody else holds it; a batch whose tables find no room takes nothing."""
    ctx, kv, pool = cache_of(3)
    a = kv.new_sequence()
    kv.batch(pool, [(a, 64)])
    b = kv.fork(a)
    kv.cut(a, 10), kv.cut(b, 10)
    kv.batch(pool, [(kv.new_sequence(), 64)])
    assert kv.free_pages == 1
    with pytest.raises(ValueError, match="exhausted"):
        kv.batch(gptq.ActivationArena(ctx, 256), [(a, 1), (b, 1)])
    assert kv.free_pages == 1 and kv.length(a) == 10 and kv._lists[a] == kv._lists[b] and not ctx.log
    kv.batch(pool, [(a, 1), (b, 1)])
    assert kv.free_pages == 0 and kv._lists[a] != kv._lists[b] and len(ctx.log) == 2 and kv.length(b) == 11
    c = kv.fork(kv.new_sequence())
    with pytest.raises(ValueError, match="1 pages"):
        kv.batch(pool, [(c, 1)])


def test_fork_shares_whole_pages():
    ctx, kv, pool = cache_of(6)
    a = kv.new_sequence()
    kv.batch(pool, [(a, 130)])
    b = kv.fork(a)                                                               # two whole pages shared, the third copied
    assert kv.free_pages == 2 and kv.length(b) == 130
    moves = [args for call, args in ctx.log if call == "kv_move"]
    assert [m[6] for m in moves] == [kv.page_bytes, kv.scale_bytes] and all(m[9] == 1 for m in moves)
    assert moves[0][7] == kv._lists[b][2] and moves[0][8] == kv._lists[a][2] and kv._lists[a][:2] == kv._lists[b][:2]
    kv.free(a)
    assert kv.free_pages == 3                                                    # what b holds stays
    c = kv.fork(b)
    kv.cut(c, 100)                                                               # inside a page that b holds too: copied before c appends
    ctx.log.clear()
    batch = kv.batch(pool, [(c, 5), (b, 1)])
    assert kv._lists[c][0] == kv._lists[b][0] and kv._lists[c][1] != kv._lists[b][1] and len(ctx.log) == 2
    assert list(tables(batch)[1]) == [105, 131]
    kv.free(b), kv.free(c)
    assert kv.free_pages == 6 and kv._users == [0] * 6
    full = kv.new_sequence()
    kv.batch(pool, [(full, 6 * 64 - 1)])
    with pytest.raises(ValueError, match="no page"):
        kv.fork(full)
    kv.batch(pool, [(full, 1)])
    kv.fork(full)                                                                # nothing but whole pages


def test_arguments():
    ctx, kv, pool = cache_of(4)
    arena = pool.arena
    C, KVD = CFG.n_embd, kv.row_len
    a = kv.new_sequence()
    batch = kv.batch(pool, [(a, 6)])
    q, k, v, out, h, hk, short = tensors(arena, ((6, C), "f32"), ((6, KVD), "f32"), ((6, KVD), "f32"), ((6, C), "f32"), ((6, C), "f16"), ((6, KVD), "f16"), ((5, C), "f32"))
    m = model_of(ctx)
    m.loras = {}
    m.f32 = {"rope": gptq.Tensor(m.weights, 0, 256 * 64, (256, 64), "f32"), "n": gptq.Tensor(m.weights, 0, 32, (32,), "f32")}
    far, = tensors(Held(1 << 20), ((6, C), "f32"))
    for args, kw in (((q, k, hk, batch, out), {}), ((h, k, v, batch, out), {}), ((short, k, v, batch, out), {}), ((q, k, short, batch, far), {}), ((q, k, v, batch, out), {"rope": "x"}),
                     ((q, k, v, batch, out), {"q_norm": "n"}), ((q, k, v, batch, short), {})):
        with pytest.raises(ValueError):
            kv.append(0, m, *args, **kw)
    for args in ((q, h, batch), (short, out, batch), (q, far, batch), (k, out, batch)):
        with pytest.raises(ValueError):
            kv.attend(0, *args)
    assert not ctx.log
    kv.append(1, m, q, k, v, batch, h)
    kv.attend(1, h, h, batch)
    (c1, a1), (c2, a2) = ctx.log
    assert (c1, c2) == ("paged_append", "paged_attention") and a1[7] == 6 and a1[9] == a2[2] == ql.DTYPE_F16
    desc = a2[4]
    assert (desc.k_off, desc.v_off, desc.k_scale_off, desc.v_scale_off) == (kv.regions[2], kv.regions[3], kv.scales[2], kv.scales[3])
    # adapters
    m.linears = {"w": gptq._Linear(None, 64, 32)}
    m._place = lambda d: 0
    good = (np.zeros((3, 8, 64)), np.zeros((3, 32, 8)))
    for a_, b_, s in ((good[0][:, :, :60], good[1], None), (good[0], good[1][:2], None), (good[0], good[1], np.ones(2)), (np.zeros((3, 12, 64)), np.zeros((3, 32, 12)), None)):
        with pytest.raises(ValueError, match="lora"):
            m.upload_lora("w", a_, b_, s)
    with pytest.raises(ValueError, match="missing"):
        m.upload_lora("x", *good)
    m.upload_lora("w", *good)
    with pytest.raises(ValueError, match="already"):
        m.upload_lora("w", *good)
    x, c, ids, wide = tensors(arena, ((6, 64), "f32"), ((6, 32), "f32"), ((6,), "i32"), ((6, 32), "f16"))
    for args in ((x, ["v"], ids, [c], 6), (x, ["w"], ids, [c, c], 6), (x, ["w"], c, [c], 6), (x, ["w"], ids, [wide], 6), (x, ["w"], ids, [c], 7), (far, ["w"], ids, [c], 6)):
        with pytest.raises(ValueError):
            m.lora_add(*args)
    ctx.log.clear()
    m.lora_add(x, ["w"], ids, [c], 6)
    call, args = ctx.log[0]
    assert call == "lora_add" and args[7] == args[8] == [c.offset] and args[4] == [x.offset]


class Served(Model):
    """test_draft's model with adapters on q, k, v and o, and passes over several sequences."""

    def __init__(self, ctx, n=3, rank=8):
        super().__init__(ctx)
        C, KVD, g = CFG.n_embd, gptq.qwen_kv_dim(CFG), np.random.default_rng(21)
        self.adapters = {}
        for layer in range(CFG.n_layer):
            for name, N in (("q", C), ("k", KVD), ("v", KVD), ("o", C)):
                a, b = ((g.standard_normal(s) * 0.05).astype(np.float16) for s in ((n, rank, C), (n, N, rank)))
                scale = g.uniform(0.5, 2, n).astype(np.float32)
                self.gpu.upload_lora(f"L{layer}.{name}", a, b, scale)
                self.adapters[layer, name] = scale[:, None, None] * b.astype(np.float64) @ a.astype(np.float64)

    def step(self, pool, kv, batch, tokens, ids):
        """One pass over the batch's rows; logits [M, V]."""
        m, M, C, KVD = self.gpu, batch.M, CFG.n_embd, gptq.qwen_kv_dim(CFG)
        tok, who = pool.alloc((M,), "u32"), pool.alloc((M,), "i32")
        tok.write(np.asarray(tokens, np.uint32)), who.write(np.asarray(ids, np.int32))
        h = pool.alloc((M, C))
        m.embed(tok, h, M)
        for layer in range(CFG.n_layer):
            L = f"L{layer}."
            n, q, k, v, a, o = (pool.alloc((M, w)) for w in (C, C, KVD, KVD, C, C))
            m.rmsnorm(h, L + "in", n, M, C, 1e-6)
            m.gemm_batch(n, [L + "q", L + "k", L + "v"], [q, k, v], M)
            m.lora_add(n, [L + "q", L + "k", L + "v"], who, [q, k, v], M)
            kv.append(layer, m, q, k, v, batch, q, q_norm=L + "qn", k_norm=L + "kn")
            kv.attend(layer, q, a, batch)
            m.gemm(a, L + "o", o, None, M, C, C)
            m.lora_add(a, [L + "o"], who, [o], M)
            s, n2, ga, up, act, d, h2, last = (pool.alloc((M, w)) for w in (C, C, CFG.intermediate, CFG.intermediate, CFG.intermediate, C, C, C))
            m.rmsnorm(o, L + "post", n2, M, C, 1e-6, residual=h, sum_out=s)
            m.gemm_batch(n2, [L + "gate", L + "up"], [ga, up], M)
            m.silu_mul(ga, up, act, M * CFG.intermediate)
            m.gemm(act, L + "down", d, None, M, C, CFG.intermediate)
            m.rmsnorm(d, "norm", last, M, C, 1e-6, residual=s, sum_out=h2)
            h = h2
        logits = pool.alloc((M, CFG.vocab_size))
        m.gemm(last, "embed", logits, None, M, CFG.vocab_size, C)
        out = logits.read()
        pool.reset()
        return out

    def text(self, tokens, who, dtype):
        """Logits of a whole sequence's tokens under an adapter in 64 bits, its keys and values rounded as a cache of the type holds them."""
        w, M, H, KV, D = self.w, len(tokens), CFG.n_head, CFG.n_kv_head, 64
        pos, seen = np.arange(M), np.tril(np.ones((M, M), bool))

        def cache(x):
            if dtype == "f16":
                return x.astype(np.float16).astype(np.float64)
            p = np.concatenate([np.broadcast_to(power(np.abs(x[t:t + 16]).max((0, 2), keepdims=True)), (len(x[t:t + 16]), KV, 1)) for t in range(0, M, 16)])
            return f8_decode(f8_encode(x / p)) * p

        def lin(n, layer, name):
            return n @ (w[layer, name] + (self.adapters[layer, name][who] if who >= 0 else 0)).T
        norm = lambda a, n: a / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-6) * n  # noqa: E731
        h = w["embed"][tokens].astype(np.float64)
        for layer in range(CFG.n_layer):
            n = norm(h, w[layer, "in"])
            q, k, v = (lin(n, layer, p) for p in "qkv")
            q = turned(q.reshape(M, H, D), pos, w[layer, "qn"].astype(np.float64))
            k = cache(turned(k.reshape(M, KV, D), pos, w[layer, "kn"].astype(np.float64)))
            h = h + lin(attention(q, k, cache(v.reshape(M, KV, D)), seen)[0].reshape(M, H * D), layer, "o")
            n = norm(h, w[layer, "post"])
            ga, up = n @ w[layer, "gate"].T, n @ w[layer, "up"].T
            h = h + (ga / (1 + np.exp(-ga)) * up) @ w[layer, "down"].T
        return norm(h, w["norm"]) @ w["embed"].astype(np.float64).T


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f8"])
def test_model_serves_many(ctx, dtype):
    """Prompts, single tokens and a fork of several sequences with adapters of their own, in passes of up to 16 rows (fp32-grade linears),
    against each text by itself. An e4m3 cache's values next to a border of rounding may fall to its other side, by 2^-3 of a
    value, for the linears' 2^-20: of some hundred keys and values a row, one in ten thousand."""
    model, pool = Served(ctx), gptq.ActivationArena(ctx, 16 << 20)
    kv, g = gptq.PagedKvCache(ctx, CFG, 12, 64, dtype), np.random.default_rng(4)
    tol = 2.0 ** -8 if dtype == "f16" else 2.0 ** -6
    texts, who = {}, {}

    def go(rows, pad=0):
        new = {s: [int(t) for t in g.integers(0, CFG.vocab_size, n)] for s, n in rows}
        batch = kv.batch(pool, rows, M=sum(n for _, n in rows) + pad)
        ids = [who[s] for s, n in rows for _ in range(n)] + [-1] * pad
        logits = model.step(pool, kv, batch, [t for s, _ in rows for t in new[s]] + [0] * pad, ids)
        at = 0
        for s, n in rows:
            texts[s] = texts[s] + new[s]
            if n:
                want = model.text(texts[s], who[s], dtype)[-n:]
                assert np.abs(logits[at:at + n] - want).max() <= tol * np.abs(want).max(), (s, np.abs(logits[at:at + n] - want).max() / np.abs(want).max())
            at += n

    a, b, c = (kv.new_sequence() for _ in range(3))
    for s, w in ((a, 0), (b, -1), (c, 2)):
        texts[s], who[s] = [], w
    go([(a, 7), (b, 5), (c, 3)])
    go([(c, 1), (a, 9), (b, 1)], pad=3)
    for _ in range(3):
        go([(a, 15)])
    go([(a, 1), (b, 1), (c, 1)])
    go([(a, 6), (c, 10)])                                                        # a enters its second page
    d = kv.fork(a)
    texts[d], who[d] = list(texts[a]), who[a]
    go([(a, 1), (d, 1), (b, 0), (c, 1)])
    go([(d, 4), (a, 1)])
    kv.cut(d, 60)
    texts[d] = texts[d][:60]
    go([(d, 3), (a, 1)])                                                         # within a page that both held
    kv.free(a), kv.free(d)
    go([(b, 2), (c, 12)])
    pool.arena.release(), kv.release(), model.gpu.release()
