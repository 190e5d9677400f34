"""Passes over many requests that the library always refuses: PagedKvCache refuses them itself, before it takes pages or counts tokens, in the Python host and
in the Node host."""
import dataclasses
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from tests.test_batch_hosts import CFG, Context
from webllm_amd import gptq

SCRIPT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "js", "batch_limits.js")
WIDE = dataclasses.replace(CFG, n_head=128, n_kv_head=32, n_embd=128 * 64)       # 192 heads of q, k and v a row


def cache(pages, config=CFG, page_size=256):
    ctx = Context()
    return gptq.PagedKvCache(ctx, config, pages, page_size, "f16"), gptq.ActivationArena(ctx, 1 << 24)


def state(kv):
    return kv.free_pages, dict(kv._lengths), {s: list(p) for s, p in kv._lists.items()}


def refuses(kv, pool, *args, match):
    before, used = state(kv), pool.layout.used
    with pytest.raises(ValueError, match=match):
        kv.batch(pool, *args)
    assert state(kv) == before and pool.layout.used == used


def test_rows():
    kv, pool = cache(300)
    a, b = kv.new_sequence(), kv.new_sequence()
    refuses(kv, pool, [(a, 65000), (b, 536)], match="65535 rows")
    refuses(kv, pool, [(a, 5)], 65536, match="65535 rows")
    refuses(kv, pool, [(a, 0)], 0, match="rows")
    refuses(kv, pool, [(a, 2.5)], match="whole")
    assert kv.batch(pool, [(a, 65000), (b, 535)]).M == 65535
    kv, pool = cache(300, WIDE)
    a = kv.new_sequence()
    refuses(kv, pool, [(a, 43691)], match="heads")                               # 43691 * 192 is the first above 2^23
    assert kv.batch(pool, [(a, np.int64(43690))]).M == 43690


def test_numbers_that_are_not_whole():
    kv, pool = cache(8)
    a = kv.new_sequence()
    kv.batch(pool, [(a, 9)])
    for args in (([(a, 2.0)],), ([(a, 2.5)],), ([(a, float("nan"))],), ([(a, 2)], 4.0), ([(a, None)],)):
        refuses(kv, pool, *args, match="whole")
    for tokens in (1.5, 3.0, None):
        with pytest.raises(ValueError, match="whole"):
            kv.cut(a, tokens)
    assert kv.length(a) == 9
    b = kv.batch(pool, [(a, np.int32(3))], np.int64(4))
    assert (type(b.M), type(kv.length(a)), kv.length(a), b.desc.max_rows) == (int, int, 12, 3)
    kv.cut(a, np.int64(2))
    assert (type(kv.length(a)), kv.length(a)) == (int, 2)


def test_sequences():
    kv, pool = cache(5000)
    all_ = [(kv.new_sequence(), 1) for _ in range(4097)]
    refuses(kv, pool, all_, match="4096 sequences")
    assert kv.batch(pool, all_[:4096]).desc.n_seq == 4096
    many = dataclasses.replace(CFG, n_head=2048, n_kv_head=2048, n_embd=2048 * 16)
    kv, pool = cache(5000, many)
    all_ = [(kv.new_sequence(), int(i == 0)) for i in range(2049)]
    refuses(kv, pool, all_, match="heads")                                       # 2049 * 2048 kv heads of sequences
    kv.batch(pool, all_[:2048])


def test_tokens():
    kv, pool = cache((1 << 18) + 2)
    a = kv.new_sequence()
    full = (1 << 26) - 1                                                         # as after a long text: all but one token
    kv._lists[a], kv._lengths[a] = [kv._take() for _ in range(1 << 18)], full
    refuses(kv, pool, [(a, 2)], match="tokens")
    assert kv.batch(pool, [(a, 1)]).desc.max_len == 1 << 26
    refuses(kv, pool, [(a, 1)], match="tokens")


@pytest.mark.parametrize("heads, kv, width", [(4, 2, 4 * 8), (4, 2, 4 * 24), (2, 2, 2 * 272), (4, 3, 4 * 16), (8192, 8192, 8192 * 16)])
def test_heads(heads, kv, width):
    with pytest.raises(ValueError, match="head"):
        cache(4, dataclasses.replace(CFG, n_head=heads, n_kv_head=kv, n_embd=width))


@pytest.mark.skipif(shutil.which("node") is None, reason="node not installed")
def test_node():
    r = subprocess.run([shutil.which("node"), SCRIPT], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    got = json.loads(r.stdout.strip().splitlines()[-1])
    for name, word in (("rows", "65535 rows"), ("padding", "65535 rows"), ("none", "rows"), ("wide", "heads"), ("sequences", "4096 sequences"), ("kvHeads", "heads"), ("tokens", "tokens"),
                       ("head8", "head"), ("head24", "head"), ("head272", "head"), ("headsApart", "head"), ("heads8192", "head")):
        assert got[name][0] and word in got[name][0] and got[name][1], (name, got[name])
    assert got["taken"] == [65535, 43690, 4096, 2048, 1 << 26]
