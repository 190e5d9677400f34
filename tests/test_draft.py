"""Speculative decoding through the hosts (webllm_amd.gptq and webllm_amd/js): a model's drafted pass from hidden rows to an
accepted path, in the order a program has it, and the same through Node.

The pass is compared with 64-bit arithmetic over the same weights. Its linears run in fp32 grade and its caches in fp32 (or
fp16, whose rounding is 2^-11 of a key or value); the tolerances below follow from that at each step."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from tests.test_gpu_attn_tree import formula as attention, seen_of, tree
from tests.test_gpu_logprobs import reference as logprobs
from tests.test_gpu_rope import angles, formula as rope
from webllm_amd import gptq, synth
from webllm_amd import qlinear as ql

NODE = shutil.which("node")
SCRIPT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "js", "draft_check.js")
needs_node = pytest.mark.skipif(NODE is None, reason="node not installed")
CFG = gptq.QwenConfig(vocab_size=640, block_size=256, n_layer=2, n_head=6, n_kv_head=2, n_embd=384, intermediate=512, rope_theta=1e4)


def node(*args):
    r = subprocess.run([NODE, SCRIPT, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout.strip().splitlines()[-1])


@needs_node
def test_node_masks_and_refusals():
    r = node("abi")
    assert len(r["functions"]) == 6
    masks, depths = ql.tree_masks(r["parents"])
    assert [int(w) for w in r["masks"]] == [int(w) for w in masks.reshape(-1)] and r["depths"] == list(depths)
    assert "QL_E_INVALID" in r["bad"] and "too short" in r["short"] and "too few arguments" in r["few"] and "handle" in r["noHandle"]


def turned(x, pos, norm):
    c, s = angles(pos, x.shape[-1], CFG.rope_theta)
    return rope(x, norm, 1e-6, c, s, x.shape[-1], False)[0]


@pytest.mark.gpu
@needs_node
def test_node_drafted_pass(tmp_path):
    g = np.random.default_rng(3)
    H, KV, D, past, M = CFG.n_head, CFG.n_kv_head, 64, 90, 21
    parents = tree(M, 5)
    masks, depths = ql.tree_masks(parents)
    path = [0]
    while len(path) < 4 and any(parents[m] == path[-1] for m in range(M)):
        path.append(next(m for m in range(M) if parents[m] == path[-1]))
    n = len(path)
    x = {}
    for i, rows in ((0, past), (1, M), (2, 1)):
        for name, w in (("q", H * D), ("k", KV * D), ("v", KV * D)):
            x[f"{name}{i}"] = g.standard_normal((rows, w)).astype(np.float32)
    x.update(pos0=np.arange(past, dtype=np.int32), pos1=(past + depths).astype(np.int32), pos2=np.array([past + n], np.int32),
             x=(2 * g.standard_normal((M, 700))).astype(np.float32), tok=g.integers(-1, 700, (M, 2)).astype(np.int32), path=np.array(path, np.int32))
    for name, a in x.items():
        a.tofile(tmp_path / name)
    norm = (1 + 0.2 * g.standard_normal(D)).astype(np.float32)
    (tmp_path / "cases.json").write_text(json.dumps({
        "config": {"vocabSize": 640, "blockSize": 256, "nLayer": 2, "nHead": H, "nKvHead": KV, "nEmbd": H * D, "intermediate": 512, "ropeTheta": CFG.rope_theta},
        "M": M, "past": past, "V": 700, "parents": [int(p) for p in parents], "depths": [int(d) for d in depths], "path": n, "qn": [float(v) for v in norm]}))
    errors = node("gpu", str(tmp_path))["errors"]
    heads = lambda name, h: x[name].reshape(-1, h, D)  # noqa: E731
    k = np.concatenate([turned(heads("k0", KV), x["pos0"], None), turned(heads("k1", KV), x["pos1"], None)])
    v = np.concatenate([heads("v0", KV), heads("v1", KV)])
    q1 = turned(heads("q1", H), x["pos1"], norm)
    keep = list(range(past)) + [past + m for m in path]
    k2 = np.concatenate([k[keep], turned(heads("k2", KV), x["pos2"], None)])
    v2 = np.concatenate([v[keep], heads("v2", KV)])
    q2 = turned(heads("q2", H), x["pos2"], norm)
    for dtype in ("f32", "f16"):
        # the rotation's own rounding, 32 u of q and k, enters the scores (|q . k| / 8 of some 40): 2^-19 of a result of about
        # one; a half cache's half steps, 2^-11 of keys and values, some 2^-10 times the scores' size of 4
        rounded = (lambda a: a.astype(np.float16).astype(np.float64)) if dtype == "f16" else (lambda a: a.astype(np.float64))
        for name, qq, kk, vv, seen in (("o", q1, k, v, seen_of(masks, M, past)), ("o2", q2, k2, v2, np.ones((1, past + n + 1), bool))):
            want, tol = attention(qq, rounded(kk), rounded(vv), seen)
            got = np.fromfile(tmp_path / f"{name}.{dtype}", np.float32).reshape(want.shape)
            extra = 2.0 ** -17 if dtype == "f32" else 2.0 ** -8                # a key on the other side of an fp16 border moves by a step
            assert (np.abs(got - want) <= tol + extra).all(), (name, dtype, np.abs(got - want).max())
        lp, ent, ids, tlp = logprobs(x["x"], x["tok"], 3)
        assert np.abs(np.fromfile(tmp_path / f"lp.{dtype}", np.float32).reshape(lp.shape) - lp).max() < 1e-5
        assert np.abs(np.fromfile(tmp_path / f"ent.{dtype}", np.float32) - ent).max() < 1e-4
        assert np.array_equal(np.fromfile(tmp_path / f"ids.{dtype}", np.int32).reshape(ids.shape), ids)
        assert np.abs(np.fromfile(tmp_path / f"tlp.{dtype}", np.float32).reshape(tlp.shape) - tlp).max() < 1e-5
    assert "fp16 cache" in errors["store"] and "fp16 cache" in errors["attend"] and "another type" in errors["type"]
    assert "QL_E_RANGE" in errors["range"] and "at least n" in errors["path"] and "missing f32 weight" in errors["missing"]
    assert "come with" in errors["pair"] and "dtype" in errors["dtype"]
    assert "another type" in errors["half"] and "another type" in errors["halfOut"] and "as many source offsets" in errors["regions"]


# ------------------------------------------------------------------ a model's pass, from embedding to accepted path

class Model:
    """Two layers with random GPTQ weights, and the same weights in 64 bits."""

    def __init__(self, ctx):
        C, I, KVD = CFG.n_embd, CFG.intermediate, gptq.qwen_kv_dim(CFG)
        self.gpu, self.w = gptq.QuantLinearModel(ctx, 16 << 20), {}
        g = np.random.default_rng(11)
        for layer in range(CFG.n_layer):
            for i, (name, K, N) in enumerate((("q", C, C), ("k", C, KVD), ("v", C, KVD), ("o", C, C), ("gate", C, I), ("up", C, I), ("down", I, C))):
                t = synth.gptq_linear(K, N, 128, seed=100 * layer + i)
                self.gpu.upload_gptq_linear(f"L{layer}.{name}", t.qweight, t.qzeros, t.scales, K, N, 128)
                self.w[layer, name] = self.gpu.dequantize(f"L{layer}.{name}").astype(np.float64)
            for name, size in (("in", C), ("post", C), ("qn", 64), ("kn", 64)):
                self.w[layer, name] = (1 + 0.1 * g.standard_normal(size)).astype(np.float32)
                self.gpu.upload_f32(f"L{layer}.{name}", self.w[layer, name])
        self.w["embed"] = (0.5 * g.standard_normal((CFG.vocab_size, C))).astype(np.float16)
        self.gpu.upload_f16_bits("embed", self.w["embed"].view(np.uint16), (CFG.vocab_size, C))
        self.w["norm"] = (1 + 0.1 * g.standard_normal(C)).astype(np.float32)
        self.gpu.upload_f32("norm", self.w["norm"])
        self.gpu.make_rope_table(CFG.block_size, 64, CFG.rope_theta)

    def run(self, pool, kv, tokens, positions, past, masks, chosen):
        """One pass; (logits, logprobs of chosen [M, T], entropy, top 3 ids, their logprobs)."""
        m, M, C = self.gpu, len(tokens), CFG.n_embd
        KVD = gptq.qwen_kv_dim(CFG)
        tok, pos = pool.alloc((M,), "u32"), pool.alloc((M,), "i32")
        tok.write(np.asarray(tokens, np.uint32))
        pos.write(np.asarray(positions, np.int32))
        words = None
        if masks is not None:
            words = pool.alloc(masks.shape, "u64")
            words.write(masks)
        h = pool.alloc((M, C))
        m.embed(tok, h, M)
        for layer in range(CFG.n_layer):
            L = f"L{layer}."
            n, q, k, v, a, o = (pool.alloc((M, w)) for w in (C, C, KVD, KVD, C, C))
            m.rmsnorm(h, L + "in", n, M, C, 1e-6)
            m.gemm(n, L + "q", q, None, M, C, C)
            m.gemm(n, L + "k", k, None, M, KVD, C)
            m.gemm(n, L + "v", v, None, M, KVD, C)
            kv.rotate_store(layer, m, q, k, v, pos, q, M, past, q_norm=L + "qn", k_norm=L + "kn")
            kv.attend_tree(layer, q, a, M, past, words)
            m.gemm(a, L + "o", o, None, M, C, C)
            s, n2, ga, up, act, d, h2 = (pool.alloc((M, w)) for w in (C, C, CFG.intermediate, CFG.intermediate, CFG.intermediate, C, C))
            m.rmsnorm(o, L + "post", n2, M, C, 1e-6, residual=h, sum_out=s)
            m.gemm(n2, L + "gate", ga, None, M, CFG.intermediate, C)
            m.gemm(n2, L + "up", up, None, M, CFG.intermediate, C)
            m.silu_mul(ga, up, act, M * CFG.intermediate)
            m.gemm(act, L + "down", d, None, M, C, CFG.intermediate)
            unused = pool.alloc((M, C))
            m.rmsnorm(d, "norm", unused, M, C, 1e-6, residual=s, sum_out=h2)
            h = h2
        n = unused
        logits = pool.alloc((M, CFG.vocab_size))
        m.gemm(n, "embed", logits, None, M, CFG.vocab_size, C)
        chosen = np.asarray(chosen, np.int32).reshape(M, -1)
        t, lp, ent = pool.alloc(chosen.shape, "i32"), pool.alloc(chosen.shape), pool.alloc((M,))
        ids, tlp = pool.alloc((M, 3), "i32"), pool.alloc((M, 3))
        t.write(chosen)
        m.token_logprobs(logits, M, CFG.vocab_size, t, lp, ent, ids, tlp)
        out = [x.read() for x in (logits, lp, ent, ids, tlp)]
        pool.reset()
        return out

    def plain(self, tokens, positions, seen, half):
        """Logits of rows that see each other as `seen` says, in 64 bits (a half cache's keys and values rounded)."""
        w, M, H, KV, D = self.w, len(tokens), CFG.n_head, CFG.n_kv_head, 64
        cache = (lambda a: a.astype(np.float16).astype(np.float64)) if half else (lambda a: a)
        norm = lambda a, n: a / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-6) * n  # noqa: E731
        h = w["embed"][tokens].astype(np.float64)
        for layer in range(CFG.n_layer):
            n = norm(h, w[layer, "in"])
            q, k, v = (n @ w[layer, p].T for p in ("q", "k", "v"))
            q = turned(q.reshape(M, H, D), positions, w[layer, "qn"].astype(np.float64))
            k = cache(turned(k.reshape(M, KV, D), positions, w[layer, "kn"].astype(np.float64)))
            a = attention(q, k, cache(v.reshape(M, KV, D)), seen)[0].reshape(M, H * D)
            h = h + a @ w[layer, "o"].T
            n = norm(h, w[layer, "post"])
            ga, up = n @ w[layer, "gate"].T, n @ w[layer, "up"].T
            h = h + (ga / (1 + np.exp(-ga)) * up) @ w[layer, "down"].T
        return norm(h, w["norm"]) @ w["embed"].astype(np.float64).T


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_model_drafts_and_accepts(ctx, dtype):
    """A prompt, a drafted tree, its accepted path, and the next token: logits as if the accepted tokens had been the text all
    along, in the cache and in one forked from it. Rows of up to 16 run the fp32-grade linears: what is left is some 2^-20 of
    a logit per linear, and with a half cache its keys' and values' rounding of 2^-11."""
    model, pool = Model(ctx), gptq.ActivationArena(ctx, 16 << 20)
    kv, other = gptq.KvCache(ctx, CFG, dtype), gptq.KvCache(ctx, CFG, dtype)
    half, g = dtype == "f16", np.random.default_rng(4)
    tol = 2.0 ** -8 if half else 2.0 ** -15

    def close(got, want, scale=1.0):
        assert np.abs(got - want).max() <= tol * scale * np.abs(want).max(), (np.abs(got - want).max(), np.abs(want).max())

    text = [int(t) for t in g.integers(0, CFG.vocab_size, 29)]
    for at in range(0, 29, 13):                                              # the prompt in pieces of up to 13 rows, causal
        piece = text[at:at + 13]
        got = model.run(pool, kv, piece, range(at, at + len(piece)), at, None, [[0]] * len(piece))
        want = model.plain(text[:at + len(piece)], np.arange(at + len(piece)), np.tril(np.ones((at + len(piece),) * 2, bool)), half)
        close(got[0], want[at:])
    past, M = len(text), 14
    parents = np.array([-1, -1, 0, 0, 1, 2, 2, 3, 5, 5, 6, 8, 8, 9], np.int32)
    masks, depths = ql.tree_masks(parents)
    drafted = [int(t) for t in g.integers(0, CFG.vocab_size, M)]
    children = [[m for m in range(M) if parents[m] == n] for n in range(M)]
    width = max(1, max(len(c) for c in children))
    chosen = [[drafted[m] for m in c] + [-1] * (width - len(c)) for c in children]
    got = model.run(pool, kv, drafted, past + depths, past, masks, chosen)
    seen = np.zeros((past + M,) * 2, bool)
    seen[:past, :past] = np.tril(np.ones((past, past), bool))
    seen[past:] = seen_of(masks, M, past)
    want = model.plain(text + drafted, np.concatenate([np.arange(past), past + depths]), seen, half)[past:]
    close(got[0], want)
    lp, ent, _, _ = logprobs(got[0], np.array(chosen), 3)                    # of the logits that the pass made
    assert np.abs(got[1] - lp).max() < 1e-5 and np.abs(got[2] - ent).max() < 1e-4
    order = np.argsort(-got[0], 1, kind="stable")[:, :3]
    assert np.array_equal(got[3], order)
    path = [0]
    while children[path[-1]]:                                                # the most likely drafted continuation
        path.append(max(children[path[-1]], key=lambda m: got[1][path[-1], children[path[-1]].index(m)]))
    assert len(path) >= 3 and path != list(range(len(path)))
    rows = pool.alloc((len(path),), "i32")
    rows.write(np.array(path, np.int32))
    kv.accept(past, rows, len(path))
    ctx.sync()
    pool.reset()
    accepted = text + [drafted[m] for m in path]
    kv.fork(other, len(accepted))
    for cache, token in ((kv, 17), (other, 400)):
        n = len(accepted)
        got = model.run(pool, cache, [token], [n], n, None, [[token]])
        want = model.plain(accepted + [token], np.arange(n + 1), np.tril(np.ones((n + 1, n + 1), bool)), half)
        close(got[0], want[-1:])
    kv.release()
    other.release()
    model.gpu.release()


@pytest.mark.gpu
def test_host_refusals(ctx):
    kv, half = gptq.KvCache(ctx, CFG), gptq.KvCache(ctx, CFG, "f16")
    pool = gptq.ActivationArena(ctx, 4 << 20)
    model = gptq.QuantLinearModel(ctx, 1 << 20)
    C, KVD = CFG.n_embd, gptq.qwen_kv_dim(CFG)
    q, k, o, pos, words = pool.alloc((4, C)), pool.alloc((4, KVD)), pool.alloc((4, C)), pool.alloc((4,), "i32"), pool.alloc((4, 1), "u64")
    with pytest.raises(ValueError, match="missing rope table"):
        kv.rotate_store(0, model, q, k, k, pos, o, 4, 0)
    model.make_rope_table(64, 64, 1e4)
    with pytest.raises(ValueError, match="already exists"):
        model.make_rope_table(64, 64, 1e4)
    with pytest.raises(ValueError, match="exhausted"):
        model.make_rope_table(1 << 20, 64, 1e4, "big")
    bad = [lambda: gptq.KvCache(ctx, CFG, "bf16"), lambda: half.store(0, k, k, 4, 0), lambda: half.attend(0, q, o, 4, 0),
           lambda: kv.rotate_store(0, model, q, k, k, words, o, 4, 0), lambda: kv.rotate_store(0, model, q, k, k, pos, o, 5, 0),
           lambda: kv.rotate_store(0, model, q, k, k, pos, o, 4, 0, k_norm="nothing"), lambda: kv.attend_tree(0, q, o, 4, 0, pos),
           lambda: kv.attend_tree(0, q, o, 5, 0), lambda: kv.attend_tree(9, q, o, 4, 0), lambda: kv.accept(0, words, 1), lambda: kv.accept(0, pos, 5),
           lambda: kv.fork(half, 3), lambda: model.token_logprobs(q, 4, C, tokens=pos), lambda: model.token_logprobs(q, 4, C + 1, entropy=o),
           lambda: model.token_logprobs(q, 4, C, top_ids=o, top_logprobs=o)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ql.QlError):
        kv.attend_tree(0, q, o, 4, CFG.block_size - 3)
    with pytest.raises(ql.QlError):
        kv.rotate_store(0, model, q, k, k, pos, o, 4, CFG.block_size - 3)
    for x in (kv, half, pool.arena, model):
        x.release()


@pytest.mark.gpu
def test_types_of_a_drafted_pass(ctx):
    """Tensors of another type than the calls read and write are refused before anything runs."""
    kv, pool, model = gptq.KvCache(ctx, CFG), gptq.ActivationArena(ctx, 4 << 20), gptq.QuantLinearModel(ctx, 1 << 20)
    C, KVD = CFG.n_embd, gptq.qwen_kv_dim(CFG)
    q, k, o, pos, half, word = (pool.alloc(s, t) for s, t in (((4, C), "f32"), ((4, KVD), "f32"), ((4, C), "f32"), ((4,), "i32"), ((4, C), "f16"), ((4, C), "u32")))
    model.make_rope_table(64, 64, 1e4)
    model.f32["line"] = gptq.Tensor(model.weights, 0, 64, (64,), "f32")
    bad = [lambda: kv.rotate_store(0, model, half, k, k, pos, o, 4, 0), lambda: kv.rotate_store(0, model, q, half, k, pos, o, 4, 0),
           lambda: kv.rotate_store(0, model, q, k, word, pos, o, 4, 0), lambda: kv.rotate_store(0, model, q, k, k, pos, half, 4, 0),
           lambda: kv.rotate_store(0, model, q, k, k, pos, o, 4, 0, rope="line"), lambda: kv.attend_tree(0, half, o, 4, 0),
           lambda: kv.attend_tree(0, q, half, 4, 0), lambda: model.token_logprobs(q, 4, C, entropy=half),
           lambda: model.token_logprobs(q, 4, C, tokens=pos, logprobs=half), lambda: model.token_logprobs(q, 0, C, tokens=pos, logprobs=o)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for x in (kv, pool.arena, model):
        x.release()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_captured_pass(ctx, dtype):
    """A pass's operators captured once and replayed on new inputs, between the context's own calls of other sizes: the same bits
    as uncaptured, in the outputs and in the cache."""
    g, C, KVD, past, M, V = np.random.default_rng(6), CFG.n_embd, gptq.qwen_kv_dim(CFG), 170, 9, 3000
    model, pool = gptq.QuantLinearModel(ctx, 1 << 20), gptq.ActivationArena(ctx, 8 << 20)
    model.make_rope_table(CFG.block_size, 64, 1e4)
    parents = tree(M, 2)
    masks, depths = ql.tree_masks(parents)
    a, b = (gptq.KvCache(ctx, CFG, dtype) for _ in range(2))
    context = [(pool.alloc((past, C)), pool.alloc((past, KVD)), pool.alloc((past, KVD)), pool.alloc((past,), "i32"))]
    for t in context[0][:3]:
        t.write(g.standard_normal(t.shape).astype(np.float32))
    context[0][3].write(np.arange(past, dtype=np.int32))
    q, k, v, x = pool.alloc((M, C)), pool.alloc((M, KVD)), pool.alloc((M, KVD)), pool.alloc((M, V))
    pos, words, tok, path = pool.alloc((M,), "i32"), pool.alloc(masks.shape, "u64"), pool.alloc((M, 2), "i32"), pool.alloc((3,), "i32")
    pos.write((past + depths).astype(np.int32))
    words.write(masks)
    tok.write(g.integers(0, V, (M, 2)).astype(np.int32))
    sets = [[pool.alloc(s, t) for s, t in (((M, C), "f32"), ((M, C), "f32"), ((M, 2), "f32"), ((M,), "f32"), ((M, 20), "i32"), ((M, 20), "f32"))] for _ in range(2)]

    def run(cache, out):
        for layer in range(CFG.n_layer):
            cache.rotate_store(layer, model, q, k, v, pos, out[0], M, past)
            cache.attend_tree(layer, out[0], out[1], M, past, words)
        model.token_logprobs(x, M, V, tok, out[2], out[3], out[4], out[5])
        cache.accept(past, path, 3)

    def other_work():
        b.attend_tree(0, context[0][0], pool_out, past, 0)
        model.token_logprobs(x, M - 1, V, entropy=sets[1][3])

    pool_out = pool.alloc((past, C))
    for cache in (a, b):
        for layer in range(CFG.n_layer):
            cache.rotate_store(layer, model, context[0][0], *context[0][1:], pool_out, past, 0)
    ctx.graph_begin()
    run(a, sets[0])
    graph = ctx.graph_end()
    for i in range(4):
        for t in (q, k, v, x):
            t.write((2 * g.standard_normal(t.shape)).astype(np.float32))
        path.write(np.array([[0, 2, 5], [1, 3, 8], [4, 4, 0], [8, 7, 6]][i], np.int32))
        other_work()
        graph.launch()
        other_work()
        run(b, sets[1])
        ctx.sync()
        for s, t in zip(*sets):
            assert np.array_equal(s.read(), t.read(), equal_nan=True)
        rows = [c.arena.read(0, (2 * CFG.n_layer, c.region), np.uint8)[:, :(past + M) * c.row_bytes] for c in (a, b)]
        assert np.array_equal(*rows)
    graph.destroy()
    for r in (a, b, model):
        r.release()
    pool.arena.release()
