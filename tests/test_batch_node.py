"""Passes over many requests through the Node host (webllm_amd/js): sequences' pages and refusals on the CPU, and on the GPU the same
passes as the Python host's, to the bit."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from tests.test_draft import CFG
from webllm_amd import gptq
from webllm_amd import qlinear as ql

NODE = shutil.which("node")
SCRIPT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "js", "batch_check.js")
pytestmark = pytest.mark.skipif(NODE is None, reason="node not installed")


def node(*args):
    r = subprocess.run([NODE, SCRIPT, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout.strip().splitlines()[-1])


def test_node_pages_and_refusals():
    r = node("host")
    assert r["functions"] == ["loraAdd", "pagedAppend", "pagedAttention"]
    assert {"ql_lora_add", "ql_paged_append", "ql_paged_attention"} <= set(ql.header_functions())
    one = r["one"]
    start, lens, pages = one["tables"]
    assert start == [0, 70, 71] and lens == [70, 1] and len(set(pages[:3])) == 3 and pages[3] == -1 and (one["M"], one["rows"], one["free"]) == (80, 71, 3)
    d = one["desc"]
    assert (d["nSeq"], d["maxPages"], d["maxRows"], d["maxLen"]) == (2, 2, 70, 70)
    assert all(r["refused"]), r["refused"]
    assert r["kept"] == [70, 1, 3]                                               # a refused batch takes nothing
    assert r["shared"] == [2, 128, True] and r["after"] == [2, 5]
    d = r["desc"]
    assert (d["nPage"], d["pageSize"], d["nKvHead"], d["D"], d["cacheDtype"]) == (6, 64, 2, 64, ql.DTYPE_F8) and d["kOff"] < d["vOff"] < d["kScaleOff"] < d["vScaleOff"]
    assert all(r["calls"]) and all(r["lora"]) and not any("handle" in e for e in r["calls"] + r["lora"]), (r["calls"], r["lora"])
    assert all("qlinear handle" in e for e in r["library"][:3]) and "too few" in r["library"][3], r["library"]   # past the host's checks, to the library


@pytest.mark.gpu
def test_node_serves_as_python_does(ctx, tmp_path):
    g = np.random.default_rng(6)
    C, KVD, D = CFG.n_embd, gptq.qwen_kv_dim(CFG), 64
    passes = [{"rows": [[0, 70], [1, 3]], "M": 75}, {"rows": [[1, 1], [0, 1]], "M": 2}, {"rows": [[2, 1], [0, 1], [1, 40]], "M": 42, "fork": 0}, {"rows": [[2, 5], [0, 2]], "M": 7, "cut": [2, 60]}]
    norm = (1 + 0.2 * g.standard_normal(D)).astype(np.float32)
    a, b = ((g.standard_normal(s) * 0.1).astype(np.float16) for s in ((3, 8, C), (3, 128, 8)))
    scale = [0.5, 1.25, 2.0]
    a.tofile(tmp_path / "A"), b.tofile(tmp_path / "B")
    x = {}
    for i, p in enumerate(passes):
        for n, w in (("q", C), ("k", KVD), ("v", KVD)):
            x[f"{n}{i}"] = g.standard_normal((p["M"], w)).astype(np.float32)
        x[f"ids{i}"] = g.integers(-1, 4, p["M"]).astype(np.int32)
    for n, v in x.items():
        v.tofile(tmp_path / n)
    (tmp_path / "cases.json").write_text(json.dumps({
        "config": {"vocabSize": 640, "blockSize": 256, "nLayer": 2, "nHead": CFG.n_head, "nKvHead": CFG.n_kv_head, "nEmbd": C, "intermediate": 512, "ropeTheta": CFG.rope_theta},
        "passes": passes, "qn": [float(v) for v in norm], "scale": scale}))
    node("gpu", str(tmp_path))
    model = gptq.QuantLinearModel(ctx, 4 << 20)
    model.make_rope_table(256, D, CFG.rope_theta)
    model.upload_f32("qn", norm)
    model.linears["w"] = gptq._Linear(None, C, 128)
    model.upload_lora("w", a, b, scale)
    pool = gptq.ActivationArena(ctx, 8 << 20)
    for dtype in ("f16", "f8"):
        kv = gptq.PagedKvCache(ctx, CFG, 12, 64, dtype)
        seqs = [kv.new_sequence(), kv.new_sequence()]
        for i, p in enumerate(passes):
            if "fork" in p:
                seqs.append(kv.fork(seqs[p["fork"]]))
            if "cut" in p:
                kv.cut(seqs[p["cut"][0]], p["cut"][1])
            batch = kv.batch(pool, [(seqs[s], n) for s, n in p["rows"]], M=p["M"])
            q, k, v, ids, y = (pool.alloc(x[n].shape, "i32" if n.startswith("ids") else "f32") for n in (f"q{i}", f"k{i}", f"v{i}", f"ids{i}", f"v{i}"))
            for t, n in ((q, "q"), (k, "k"), (v, "v"), (ids, "ids"), (y, "v")):
                t.write(x[f"{n}{i}"])
            out = pool.alloc((p["M"], C))
            out.write(np.zeros((p["M"], C), np.float32))
            kv.append(1, model, q, k, v, batch, q, q_norm="qn")
            kv.attend(1, q, out, batch)
            model.lora_add(out, ["w"], ids, [y], p["M"])
            for n, t in (("o", out), ("y", y)):
                got, want = np.fromfile(tmp_path / f"{n}{i}.{dtype}", np.uint32), t.read()
                assert want.any() and np.array_equal(got, want.view(np.uint32).reshape(-1)), (n, i, dtype)
            pool.reset()
        kv.release()
    pool.arena.release(), model.release()
