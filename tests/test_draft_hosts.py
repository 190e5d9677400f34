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
