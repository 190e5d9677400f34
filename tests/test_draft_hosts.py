"""What the hosts of speculative decoding (webllm_amd.gptq, webllm_amd/js) make of their arguments: on the CPU with a context that
records its calls in place of the device's, and on the GPU with buffers that are kept for the largest pass."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from webllm_amd import gptq
from webllm_amd import qlinear as ql

NODE = shutil.which("node")
SCRIPT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "js", "draft_hosts_check.js")
needs_node = pytest.mark.skipif(NODE is None, reason="node not installed")


def node(*args):
    r = subprocess.run([NODE, SCRIPT, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout.strip().splitlines()[-1])


class Recorder:
    """A context that notes its calls."""

    def __init__(self, log, name="a"):
        self.log, self.name = log, name

    def __getattr__(self, call):
        return lambda *args: self.log.append((self.name, call, args))


class Memory:
    """An arena without memory."""

    def __init__(self, size=1 << 30):
        self.size = size


def tensors(arena, *specs):
    """Tensors (shape, dtype) one after the other."""
    out, at = [], 0
    for shape, dtype in specs:
        n = int(np.prod(shape))
        out.append(gptq.Tensor(arena, at, n, tuple(shape), dtype))
        at += 256 * (n * 8 // 256 + 1)
    return out


def model_of(ctx):
    m = gptq.QuantLinearModel.__new__(gptq.QuantLinearModel)
    m.ctx, m.weights, m.layout, m.linears, m.f32, m.f16 = ctx, Memory(), ql.ArenaLayout(), {}, {}, {}
    return m


def test_widths_of_logprobs():
    """T and k are the tensors' own row width, whatever number of rows they have room for."""
    log, arena = [], Memory()
    m = model_of(Recorder(log))
    x, tok, lp, ent, ids, tlp, one, lp1, flat, lpf = tensors(arena, ((256, 100), "f32"), ((256, 4), "i32"), ((256, 4), "f32"), ((256,), "f32"),
                                                             ((256, 5), "i32"), ((256, 5), "f32"), ((24,), "i32"), ((24, 1), "f32"),
                                                             ((512,), "i32"), ((1024,), "f32"))
    for M in (256, 128, 100, 3):
        m.token_logprobs(x, M, 100, tok, lp, ent, ids, tlp)
        args = log.pop()[2]
        assert (args[3], args[6], args[7]) == (M, 4, 5)
    m.token_logprobs(x, 24, 100, one, lp1)                                  # one value a row
    assert log.pop()[2][6:8] == (1, 0)
    m.token_logprobs(x, 256, 100, tok, lpf)                                 # a result without rows of its own is dense
    assert log.pop()[2][6:8] == (4, 0)
    few, ids4, three = tensors(arena, ((3, 4), "i32"), ((256, 4), "i32"), ((256, 3), "f32"))
    for kw in (dict(tokens=few, logprobs=lp, entropy=ent), dict(tokens=flat, logprobs=lpf), dict(tokens=one, logprobs=lp1), dict(tokens=tok, logprobs=three),
               dict(top_ids=ids4, top_logprobs=tlp), dict(top_ids=ids, top_logprobs=lp), dict(tokens=tok, logprobs=lp1)):
        with pytest.raises(ValueError, match="token_logprobs"):
            m.token_logprobs(x, 128, 100, **kw)
    assert log == []


@needs_node
def test_node_widths_of_logprobs():
    r = node("widths")
    assert all("qlinear handle" in e for e in r["taken"]), r["taken"]        # past the host's checks, to the library
    assert all(e and e.startswith("tokenLogprobs:") for e in r["refused"]), r["refused"]


def cache_of(ctx, log, n_head=2, n_kv_head=1):
    """A KvCache whose context only notes what it is asked for."""
    cfg = gptq.QwenConfig(vocab_size=64, block_size=32, n_layer=2, n_head=n_head, n_kv_head=n_kv_head, n_embd=128, intermediate=64, rope_theta=1e4)
    c = gptq.KvCache(ctx, cfg)
    log.clear()
    return c


def test_fork_between_contexts_is_ordered():
    """Each context has a stream of its own: nothing of the other's may still use the cache when the copy begins, and the copy is
    done when the other may use it again. On one context its stream's order is enough."""
    log = []
    one, two = Recorder(log, "one"), Recorder(log, "two")
    a, b, c = cache_of(one, log), cache_of(two, log), cache_of(one, log)
    a.fork(b, 5)
    calls = [(name, call) for name, call, _ in log]
    copy = calls.index(("one", "kv_move"))
    assert ("two", "sync") in calls[:copy] and ("one", "sync") in calls[copy:] and calls.count(("one", "kv_move")) == 1
    log.clear()
    a.fork(c, 5)
    assert [(name, call) for name, call, _ in log] == [("one", "kv_move")]


def test_fork_between_contexts_refuses_before_it_copies():
    """A context that is being captured cannot be waited for: nothing is recorded."""
    log = []

    class Capturing(Recorder):
        def sync(self):
            raise ql.QlError(-14, "ql_sync during graph capture")
    a, b = cache_of(Capturing(log, "one"), log), cache_of(Recorder(log, "two"), log)
    for x, y in ((a, b), (b, a)):
        with pytest.raises(ql.QlError):
            x.fork(y, 5)
    assert not any(call == "kv_move" for _, call, _ in log)


def test_fork_between_other_heads():
    """One head of 64 and two of 32 have rows of the same bytes, which mean other keys."""
    log = []
    ctx = Recorder(log)
    a, b = cache_of(ctx, log), cache_of(ctx, log, n_head=4, n_kv_head=2)
    assert a.row_len == b.row_len
    for x, y in ((a, b), (b, a)):
        with pytest.raises(ValueError, match="heads"):
            x.fork(y, 3)
    assert log == []


@needs_node
def test_node_fork_between_contexts_is_ordered():
    r = node("fork")
    assert "heads" in r["heads"]
    assert sorted(r["before"]) == ["one", "two"] and r["same"] == []


@needs_node
def test_node_parents_that_are_no_rows():
    """What an Int32Array would wrap or round to a row, and arrays of other kinds at the addon."""
    r = node("trees")
    assert all(e and "QL_E_INVALID" in e for e in r["refused"]), r["refused"]
    assert all(e and "expected a" in e for e in r["kinds"]), r["kinds"]
    assert r["masks"] == ["1", "3", "5", "11"] and r["depths"] == [0, 1, 1, 2]


@needs_node
def test_every_addon_function_is_a_declared_one():
    """The addon's functions, those of a drafted pass among them (which are not enumerable), and the C functions they forward to."""
    from tests.test_node_host import BINDING

    draft = {"ropeTable": "ql_rope_table", "qkNormRope": "ql_qk_norm_rope", "treeMasks": "ql_tree_masks", "attentionTree": "ql_attention_tree",
             "tokenLogprobs": "ql_token_logprobs", "kvMove": "ql_kv_move"}
    r = node("exports")
    assert r["all"] == sorted({**BINDING, **draft}) and r["hidden"] == sorted(draft)
    assert set(draft.values()) <= set(ql.header_functions())


@needs_node
def test_node_tensors_without_a_type():
    """A tensor whose type is left out, or is none of those with an array of their own, reads as fp32."""
    assert node("read") == ["Float32Array", "Float32Array", "Float32Array", "Uint16Array", "Uint32Array", "Int32Array", "BigUint64Array"]


def test_rope_table_is_a_weight():
    """Filled when the call returns, as an upload is, so that any context may read it; a refused one takes none of the arena."""
    log = []
    m = model_of(Recorder(log))
    m.weights.size = 1 << 20
    m.make_rope_table(100, 64, 1e4)
    calls = [call for _, call, _ in log]
    assert "sync" in calls[calls.index("rope_table"):] and m.f32["rope"].shape == (100, 64)
    used = m.layout.used
    with pytest.raises(ValueError, match="exhausted"):
        m.make_rope_table(1 << 20, 64, 1e4, "long")
    assert m.layout.used == used

    class Refusing(Recorder):
        def rope_table(self, *args):
            raise ql.QlError(-10, "rot_dim")
    m.ctx = Refusing(log)
    for max_pos, rot in ((100, 12), (-5, 64)):
        with pytest.raises(ql.QlError):
            m.make_rope_table(max_pos, rot, 1e4, "bad")
        assert m.layout.used == used and "bad" not in m.f32

    class Capturing(Recorder):
        def sync(self):
            raise ql.QlError(-14, "ql_sync during graph capture")
    log.clear()
    m.ctx = Capturing(log)
    with pytest.raises(ql.QlError):
        m.make_rope_table(100, 64, 1e4, "late")
    assert m.layout.used == used and not log


@needs_node
def test_node_rope_table_is_a_weight():
    r = node("table")
    assert r["used"] == [256, 256, 256] and "exhausted" in r["long"] and "handle" in r["bad"] and r["syncs"] >= 1


@pytest.mark.gpu
def test_weights_after_a_refused_table(ctx):
    model = gptq.QuantLinearModel(ctx, 1 << 16)
    with pytest.raises(ValueError, match="exhausted"):
        model.make_rope_table(1 << 16, 64, 1e4)
    with pytest.raises(ql.QlError):
        model.make_rope_table(64, 12, 1e4)
    model.make_rope_table(64, 64, 1e4)
    model.upload_f32("w", np.arange(64, dtype=np.float32))
    t = model.f32["rope"].read()
    assert np.abs(t[:, 0] - np.cos(np.arange(64))).max() < 1e-6 and np.array_equal(model.f32["w"].read(), np.arange(64, dtype=np.float32))
    model.release()


@pytest.mark.gpu
def test_fork_between_contexts(ql):
    """A prefix copied into another context's cache, whose own stream reads it at once."""
    g, a, b = np.random.default_rng(8), ql.Context(0), ql.Context(0)
    cfg = gptq.QwenConfig(vocab_size=64, block_size=2048, n_layer=3, n_head=4, n_kv_head=2, n_embd=256, intermediate=64, rope_theta=1e4)
    one, two = gptq.KvCache(a, cfg), gptq.KvCache(b, cfg)
    for layer in range(cfg.n_layer):
        for off in one.offsets(layer):
            one.arena.write(off, g.standard_normal((2048, 128)).astype(np.float32))
    pool, own = gptq.ActivationArena(b, 1 << 20), gptq.ActivationArena(a, 1 << 20)
    q, o, q1, o1 = pool.alloc((4, 256)), pool.alloc((4, 256)), own.alloc((4, 256)), own.alloc((4, 256))
    x = g.standard_normal((4, 256)).astype(np.float32)
    q.write(x)
    q1.write(x)
    one.attend_tree(2, q1, o1, 4, 1500)
    want = o1.read()
    for _ in range(5):
        two.arena.write(0, np.zeros(2 * cfg.n_layer * two.region, np.uint8))
        one.fork(two, 1504)
        two.attend_tree(2, q, o, 4, 1500)
        assert np.array_equal(o.read(), want)
    a.destroy()
    b.destroy()


@pytest.mark.gpu
def test_buffers_of_more_rows(ctx):
    """Buffers of 256 rows in passes of 128 and 100: the rows lie where the tensors' shapes say."""
    g, V = np.random.default_rng(2), 500
    model, pool = gptq.QuantLinearModel(ctx, 1 << 20), gptq.ActivationArena(ctx, 4 << 20)
    x, tok, lp, ids, tlp = (pool.alloc(s, t) for s, t in (((256, V), "f32"), ((256, 4), "i32"), ((256, 4), "f32"), ((256, 5), "i32"), ((256, 5), "f32")))
    logits, tokens = (3 * g.standard_normal((256, V))).astype(np.float32), g.integers(0, V, (256, 4)).astype(np.int32)
    x.write(logits)
    tok.write(tokens)
    full = logits.astype(np.float64)
    full -= full.max(1, keepdims=True)
    full -= np.log(np.exp(full).sum(1, keepdims=True))
    for M in (128, 100):
        lp.write(np.full((256, 4), 7, np.float32))
        ids.write(np.full((256, 5), 7, np.int32))
        model.token_logprobs(x, M, V, tok, lp, top_ids=ids, top_logprobs=tlp)
        got, best = lp.read(), ids.read()
        assert np.abs(got[:M] - np.take_along_axis(full, tokens, 1)[:M]).max() < 1e-5 and (got[M:] == 7).all()
        assert np.array_equal(best[:M], np.argsort(-logits, 1, kind="stable")[:M, :5]) and (best[M:] == 7).all()
    model.release()
    pool.arena.release()


@pytest.mark.gpu
@needs_node
def test_node_buffers_of_more_rows():
    r = node("gpu")
    assert r["ids"] == [[2, 9], [2, 9], [2, 9], [-7, -7]] and r["behind"] == [7, 7]
