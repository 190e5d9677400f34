"""ql_paged_attention over e4m3 pages whose values' scales lie far apart: a row has the accuracy of the tokens that it sees, whatever scales the tokens
have that it does not see, or gives no weight."""
import numpy as np
import pytest

from tests.arena_box import Box
from tests.paged_ref import U, Batch, Cache, f8_encode, power

pytestmark = pytest.mark.gpu

# seqs, page, H, KV, D, bounds above the tables' own
SHAPES = {
    "few": ([(20, 20), (1, 33)], 64, 3, 1, 64, {}),                              # whole tiles of 16 pairs
    "ranges": ([(1, 1500), (5, 1300), (16, 130)], 64, 4, 1, 128, {}),            # blocks dealt in ranges, joined by a merge
    "tiles": ([(80, 80), (130, 200)], 128, 6, 2, 64, {}),                        # tiles of 64 pairs, whole
    "parts": ([(70, 700)], 64, 2, 1, 192, {}),                                   # in parts of their tokens
    "wide": ([(90, 90), (70, 600)], 64, 14, 2, 128, {"max_len": 512000}),        # tiles of 128 pairs, in parts
}
# exponents of the scales of a block's four groups of 16 tokens, blocks in turn; None: zeros, under the scale that ql_paged_append gives them
SCALES = {
    "up20": [[-20, 0, -1, 0], [-22, 1, 0, -2]],
    "up40": [[-40, 0, -1, 0], [0, -41, 1, 0]],
    "stairs": [[-60, -40, -20, 0], [-7, -14, -21, -28]],
    "down": [[0, -20, -40, -60], [-60, -62, -61, -70], [-30, -90, -30, -30]],
    "zeros": [[-6, None, -5, -6], [None, None, None, None], [None, -7, -6, None]],
    "edge": [[-118, 100, 60, 100], [-118, -118, 0, 90]],
}
HALF = {                                                                         # results within fp16's range
    "up20": [[-14, 6, 5, 6], [-15, 6, 4, 5]],
    "up30": [[-24, 6, 5, 6], [4, -24, 6, -10]],
    "zeros": SCALES["zeros"],
}


def caches(batch, KV, D, exps, turned_down, seed):
    """Values' scales by token group of each sequence; keys of groups far below their block's largest scale have weight, where turned_down those of
    the others have none (their scores lie 80 below)."""
    g = np.random.default_rng([seed, 5])
    c = Cache(True, batch.n_page, batch.page, KV, D, seed)
    k = g.standard_normal((batch.n_page * batch.page, KV, D))
    v, scale = c.v.reshape(-1, KV, D), c.scale["v"].reshape(-1, KV)
    for s, (_, L) in enumerate(batch.seqs):
        at = batch.places(s)
        for t0 in range(0, L, 16):
            block = exps[t0 // 64 % len(exps)]
            e = block[t0 // 16 % 4]
            grp = at[t0] // 16
            v[grp * 16:grp * 16 + 16] = f8_encode(g.standard_normal((16, KV, D)) * 100) if e is not None else 0
            scale[grp] = 2.0 ** (-120 if e is None else e)
            small = e is not None and e <= max(x for x in block if x is not None) - 7
            k[at[t0:t0 + 16], :, 0] = -80 if turned_down and not small else 0
    grouped = k.reshape(-1, 16, KV, D)
    p = power(np.abs(grouped).max((1, 3)))
    c.k = f8_encode(grouped / p[:, None, :, None]).reshape(c.k.shape)
    c.scale["k"] = p.astype(np.float32).reshape(c.scale["k"].shape)
    return c


def formula(q, cache, batch, q16):
    """(out, tolerance) in 64 bits, row by row from what the row sees"""
    H, D, KV = q.shape[1], q.shape[2], cache.KV
    G, q = H // KV, q.astype(np.float64)
    k_all, v_all = cache.values("k"), cache.values("v")
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, (n, L) in enumerate(batch.seqs):
        at = batch.places(s)
        for i in range(n):
            m, see = batch.row_start[s] + i, L - n + i + 1
            for kv in range(KV):
                k, v, x = k_all[at[:see], kv], v_all[at[:see], kv], q[m, kv * G:(kv + 1) * G]
                sc = x @ k.T / np.sqrt(D)
                p = np.exp(sc - sc.max(1, keepdims=True))
                total = p.sum(1, keepdims=True)
                w, a = p / total, np.abs(v)
                out[m, kv * G:(kv + 1) * G] = w @ v
                pv = w @ a
                # a score: fp32 sums of D products, q's parts to 2^-22 of its row's largest, the exponential's argument and value to 2^-21 of 1 + |score|
                e = (D + 8) * U * (np.abs(x) @ np.abs(k).T / np.sqrt(D)) + np.abs(x).max(1, keepdims=True) * np.abs(k).sum(1) / np.sqrt(D) * 2.0 ** -22 + \
                    2.0 ** -21 * (np.abs(sc) + 1)
                # the weights' errors, each with the sum's; P's parts to 2^-22 of a weight; sums of blocks
                t = 2 * (w * e) @ a + 2 * (w * e).sum(1, keepdims=True) * pv + (2.0 ** -20 + (see / 32 + 64) * U) * pv
                # P's last part ends at 2^-25, half fp16's smallest step, of 2^8 P: 2^-33 of the largest weight, and no rounding costs more than the value
                # itself. A sum's steps in fp32's smallest range
                t += np.minimum(p, 2.0 ** -33) @ a / total + see * 2.0 ** -149
                if q16:                                                          # P and the result are rounded once more, the result's range ends at 2^-25
                    t += 2.0 ** -11 * (pv + np.abs(out[m, kv * G:(kv + 1) * G])) + 2.0 ** -25
                tol[m, kv * G:(kv + 1) * G] = t
    return out, tol


def run(ql, ctx, batch, H, cache, q, q16, bounds):
    box = Box(ql, ctx)
    box.put("q", q)
    box.put("out", np.zeros(q.shape, q.dtype))
    batch.put(box), cache.put(box)
    box.place()
    ctx.paged_attention(box.arena, box.off("q"), ql.DTYPE_F16 if q16 else ql.DTYPE_F32, box.arena, cache.desc(ql, box), batch.desc(ql, box, **bounds),
                        batch.M, H, box.off("out"))
    ctx.sync()
    got = box.get("out").astype(np.float64)
    box.release()
    return got


def check(ql, ctx, shape, exps, turned_down, q16):
    seqs, page, H, KV, D, bounds = SHAPES[shape]
    batch = Batch(seqs, page, seed=3)
    if bounds:
        batch.pages = np.pad(batch.pages, ((0, 0), (0, bounds["max_len"] // page - batch.max_pages)), constant_values=-1)
        batch.max_pages = batch.pages.shape[1]
    cache = caches(batch, KV, D, exps, turned_down, 7)
    q = np.random.default_rng(9).standard_normal((batch.M, H, D)).astype(np.float16 if q16 else np.float32)
    q[..., 0] = np.sqrt(D)
    out, tol = formula(q, cache, batch, q16)
    got = run(ql, ctx, batch, H, cache, q, q16, bounds)
    off = np.abs(got - out) / tol
    assert np.isfinite(got).all() and off.max() <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape), np.unique(np.nonzero(off > 1)[0])[:20])


@pytest.mark.parametrize("turned_down", [False, True])
@pytest.mark.parametrize("scales", SCALES)
@pytest.mark.parametrize("shape", SHAPES)
def test_fp32_rows(ql, ctx, shape, scales, turned_down):
    check(ql, ctx, shape, SCALES[scales], turned_down, False)


@pytest.mark.parametrize("turned_down", [False, True])
@pytest.mark.parametrize("scales", HALF)
@pytest.mark.parametrize("shape", SHAPES)
def test_fp16_rows(ql, ctx, shape, scales, turned_down):
    check(ql, ctx, shape, HALF[scales], turned_down, True)


@pytest.mark.parametrize("q16", [False, True])
def test_later_tokens_of_larger_values(ql, ctx, q16):
    """The first 16 rows of a prompt, which see one group, are as they are without the tokens behind it."""
    for L in (20, 80):
        batch = Batch([(L, L)], 64, seed=1)
        q = np.random.default_rng(2).standard_normal((batch.M, 3, 64)).astype(np.float16 if q16 else np.float32)
        got = [run(ql, ctx, batch, 3, caches(batch, 1, 64, [[-14, e, e, e]], False, 4), q, q16, {}) for e in (-14, 6)]
        out, tol = formula(q, caches(batch, 1, 64, [[-14, 6, 6, 6]], False, 4), batch, q16)
        for x in got:
            assert np.all(np.abs(x - out)[:16] <= tol[:16]) and x[:16].any(-1).all()
