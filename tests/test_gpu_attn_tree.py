"""GPU: attention of a tree of drafted tokens (ql_attention_tree) against the formula in 64 bits.

Rounding, in units u = 2^-24: a score's operands may enter as parts of 22 bits (4 u each), its D products are summed in fp32
(some 8 u of their absolute sum A / sqrt(D), as random signs go): 16 u A. exp turns that into a relative error, twice (it is in
the numerator and in the sum): 32 u A. The weights enter as parts of 22 bits and the sums over T keys are fp32 in blocks:
(32 + 2 sqrt(T)) u of sum p |V| / sum p."""
import numpy as np
import pytest

from tests.arena_box import Box

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def seen_of(masks, M, past):
    """[M, past + M] of mask words (None: causal)."""
    if masks is None:
        tail = np.tril(np.ones((M, M), bool))
    else:
        tail = (masks[:, np.arange(M) // 64] >> (np.arange(M) % 64).astype(np.uint64) & np.uint64(1)).astype(bool)
    return np.concatenate([np.ones((M, past), bool), tail], 1)


def formula(q, k, v, seen):
    """(out, bound) of q [M, H, D], k and v [T, KV, D]."""
    M, H, D = q.shape
    T, KV, _ = k.shape
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    out, tol = np.zeros((M, H, D)), np.zeros((M, H, D))
    with np.errstate(all="ignore"):
        for h in range(H):
            kh, vh = k[:, h // (H // KV)], v[:, h // (H // KV)]
            for m in range(M):
                s = seen[m]
                if not s.any():
                    continue
                kk, vv = kh[s], vh[s]
                score = kk @ q[m, h] / np.sqrt(D)
                if np.isnan(score).any() or (score == np.inf).any():
                    out[m, h] = np.nan
                    continue
                mx = score.max()
                p = np.exp(score - mx) if mx > -np.inf else np.full(score.shape, np.nan)
                out[m, h] = p @ vv / p.sum()
                fin = np.where(np.isfinite(kk), np.abs(kk), 0)
                a = (fin @ np.abs(q[m, h])).max() / np.sqrt(D)
                tol[m, h] = (32 * a + 32 + 2 * np.sqrt(T)) * U * (p @ np.abs(vv)) / p.sum()
    return out, tol


class Call:
    def __init__(self, ql, ctx, M, H, KV, D, past, half, masks, seed, extra=3, edit=None, q_scale=1.0):
        g = np.random.default_rng(seed)
        t = np.float16 if half else np.float32
        T, max_t = past + M, past + M + extra
        self.q = (q_scale * g.standard_normal((M, H, D))).astype(np.float32)
        self.k, self.v = (g.standard_normal((T, KV, D)).astype(t) for _ in range(2))
        if edit:
            edit(self)
        self.dims, self.masks = (M, H, KV, D, past, half), masks
        self.act, self.cache = Box(ql, ctx), Box(ql, ctx)
        self.act.put("q", self.q)
        if masks is not None:
            self.act.put("mask", masks, gap=8)
        self.act.put("out", np.full((M * H + 1, D), 7, np.float32))
        for n, a in (("k", self.k), ("v", self.v)):
            behind = np.full((extra, KV, D), np.nan, t)                       # rows behind the last one: not to be read into anything
            self.cache.put(n, np.concatenate([a, behind]))
        self.act.place()
        self.cache.place()
        self.args = (self.act.arena, self.act.off("q"), self.cache.arena, self.cache.off("k"), self.cache.off("v"),
                     ql.DTYPE_F16 if half else ql.DTYPE_F32, max_t, M, H, KV, D, past, None if masks is None else self.act.off("mask"), self.act.off("out"))

    def out(self):
        M, H, KV, D, past, half = self.dims
        o = self.act.get("out")
        assert (o[M * H:] == 7).all()
        return o[:M * H].reshape(M, H, D)

    def check(self, want=None):
        M, H, KV, D, past, half = self.dims
        if want is None:
            want = formula(self.q, self.k, self.v, seen_of(self.masks, M, past))
        got = self.out().astype(np.float64)
        ref, tol = want
        assert np.array_equal(np.isnan(got), np.isnan(ref)), (np.isnan(got).sum(), np.isnan(ref).sum())
        fine = np.isfinite(ref)
        assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
        if fine.any():
            off = np.abs(got[fine] - ref[fine]) - tol[fine]
            assert off.max() <= 0, (off.max(), np.abs(got[fine] - ref[fine]).max())
        return got

    def release(self):
        self.act.release()
        self.cache.release()


def tree(M, seed, width=0.9):
    g = np.random.default_rng(seed)
    return np.array([int(g.random() * (m + 1) * width) - 1 for m in range(M)], np.int32)


def run(ql, ctx, M, H, KV, D, past, half, masks, seed, **kw):
    c = Call(ql, ctx, M, H, KV, D, past, half, masks, seed, **kw)
    ctx.attention_tree(*c.args)
    c.check()
    c.release()


SHAPES = [
    # M, H, KV, D, past, label
    (1, 14, 2, 64, 0, "the first token"),
    (1, 1, 1, 8, 1, "the smallest head"),
    (5, 14, 2, 64, 300, "a small tree"),
    (2, 28, 4, 128, 63, "a context that ends inside a tile"),
    (3, 28, 4, 128, 64, "a whole tile"),
    (4, 28, 4, 128, 65, "one key more"),
    (16, 28, 4, 128, 1000, "an ordinary tree"),
    (64, 28, 4, 128, 500, "a mask word"),
    (65, 14, 2, 64, 129, "two words"),
    (256, 6, 2, 64, 200, "the largest tree"),
    (130, 4, 4, 128, 31, "no sharing of heads"),
    (24, 9, 3, 80, 77, "a head of 80"),
    (7, 4, 1, 256, 333, "the largest head"),
    (33, 5, 1, 40, 190, "five heads to one, a head of 40"),
    (12, 71, 1, 64, 100, "71 heads to one"),
    (1, 28, 4, 128, 6000, "one row, split keys"),
    (3, 16, 16, 96, 2500, "a head of 96, split keys"),
    (100, 2, 1, 200, 0, "no context, a head of 200"),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("M,H,KV,D,past,label", SHAPES)
def test_tree_matches_formula(ql, ctx, M, H, KV, D, past, half, label):
    print(label, flush=True)
    masks, _ = ql.tree_masks(tree(M, M + past))
    run(ql, ctx, M, H, KV, D, past, half, masks, 7 * M + past)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("M,past", [(1, 900), (6, 0), (40, 100), (129, 300), (256, 70)])
def test_causal_rows(ql, ctx, M, past, half):
    """Without a mask: rows in order. With the chain's mask the bits are the same."""
    c = Call(ql, ctx, M, 6, 2, 64, past, half, None, M)
    ctx.attention_tree(*c.args)
    got = c.check()
    masks, depths = ql.tree_masks(np.arange(-1, M - 1))
    assert np.array_equal(depths, np.arange(M))
    d = Call(ql, ctx, M, 6, 2, 64, past, half, masks, M)
    ctx.attention_tree(*d.args)
    assert np.array_equal(d.out(), got)
    c.release()
    d.release()


def test_agrees_with_decode_attention(ql, ctx):
    """A causal run is ql_attention_decode's, to the rounding of the two."""
    M, H, KV, D, past = 5, 28, 4, 128, 700
    c = Call(ql, ctx, M, H, KV, D, past, False, None, 3)
    ctx.attention_tree(*c.args)
    a = c.check()
    ctx.attention_decode(c.act.arena, c.act.off("q"), c.cache.arena, c.cache.off("k"), c.cache.off("v"), past + M, M, H, KV, D, past, c.act.off("out"))
    c.check()
    assert np.abs(a - c.out()).max() < 1e-4
    c.release()


@pytest.mark.parametrize("half", [False, True])
def test_rows_that_see_nothing_and_ignored_bits(ql, ctx, half):
    for M, past in ((5, 0), (70, 0), (70, 90)):
        words = (M + 63) // 64
        g = np.random.default_rng(M)
        masks = g.integers(0, 2**63, (M, words)).astype(np.uint64)
        masks[[0, M - 1]] = 0                                                # nothing of the tree
        masks[:, -1] |= np.uint64(1) << np.uint64(63)                        # bits from M on
        run(ql, ctx, M, 6, 2, 64, past, half, masks, 5)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("M,past", [(6, 40), (70, 130)])
def test_what_is_not_seen_adds_nothing(ql, ctx, M, past, half):
    """NaN and infinities in a drafted row: rows that do not see it are as without it, the others as the formula has it."""
    masks, _ = ql.tree_masks(tree(M, 3))
    for key in (past + 1, past + M - 1, past + M // 2):
        for what, value in (("k", np.nan), ("v", np.nan), ("v", np.inf), ("k", np.inf), ("v", -np.inf)):
            def edit(c):
                getattr(c, what)[key, :, 3] = value
            run(ql, ctx, M, 6, 2, 64, past, half, masks, 11, edit=edit)


@pytest.mark.parametrize("half", [False, True])
def test_not_finite_in_the_context(ql, ctx, half):
    masks, _ = ql.tree_masks(tree(9, 4))
    for what, value in (("k", np.nan), ("v", np.nan), ("v", np.inf), ("k", -np.inf)):
        def edit(c):
            getattr(c, what)[77, 1, 5] = value
        run(ql, ctx, 9, 4, 2, 128, 200, half, masks, 12, edit=edit)
    def infinite_query(c):
        c.q[4, 2, 7] = np.inf
    run(ql, ctx, 9, 4, 2, 128, 200, half, masks, 13, edit=infinite_query)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("past", [4, 40, 300, 3000])
def test_scores_all_minus_infinity(ql, ctx, past, half):
    """No score above -inf: the row is zero, as one that sees nothing; rows of other heads are as the formula has them."""
    M = 3
    def edit(c):
        c.q[:, 2:] = np.abs(c.q[:, 2:])
        c.k[:, 1] = -np.inf
    c = Call(ql, ctx, M, 4, 2, 64, past, half, None, 21, edit=edit)
    ctx.attention_tree(*c.args)
    want, tol = formula(c.q[:, :2], c.k[:, :1], c.v[:, :1], seen_of(None, M, past))
    got = c.out().astype(np.float64)
    assert (got[:, 2:] == 0).all()
    assert (np.abs(got[:, :2] - want) <= tol).all()
    c.release()


@pytest.mark.parametrize("half", [False, True])
def test_values_far_apart(ql, ctx, half):
    """Scores that one key decides, large and small values side by side in q, K and V."""
    M, past = 10, 500
    masks, _ = ql.tree_masks(tree(M, 9))
    g = np.random.default_rng(14)
    run(ql, ctx, M, 6, 2, 64, past, half, masks, 15, q_scale=30.0)
    def spread(c):
        for a, low in ((c.q, -12), (c.k, -12), (c.v, -14)):
            a *= np.exp2(g.integers(low, 4, a.shape)).astype(a.dtype)
    run(ql, ctx, M, 6, 2, 64, past, half, masks, 16, edit=spread)
    def columns(c):                                                          # a value's column far below the others
        c.v[:, :, 1] *= c.v.dtype.type(2.0 ** -9)
        c.k[:, :, 2] *= c.k.dtype.type(2.0 ** -9)
        c.q[:, :, 3] *= np.float32(2.0 ** -20)
        c.v[100] *= c.v.dtype.type(500)
    run(ql, ctx, M, 6, 2, 64, past, half, masks, 17, edit=columns)
    if not half:
        def wide(c):
            c.v *= np.float32(1e20)
            c.v[:, :, 0] *= np.float32(1e-38)
            c.k *= np.float32(1e15)
            c.q *= np.float32(1e-15)
        run(ql, ctx, M, 6, 2, 64, past, half, masks, 18, edit=wide)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("D", [8, 40, 64, 80, 128, 200, 256])
def test_short_contexts(ql, ctx, D, half):
    """A few blocks of keys, every head width, from the first length that has a wave for each of them on."""
    for M, past in ((1, 128), (9, 150), (9, 225), (40, 190), (1, 470), (16, 500)):
        print(D, M, past, flush=True)
        run(ql, ctx, M, 6, 2, D, past, half, ql.tree_masks(tree(M, M))[0], M + past)


@pytest.mark.parametrize("half", [False, True])
def test_scores_that_rise(ql, ctx, half):
    """Scores that rise along the context, slowly and by leaps, and fall: the largest is met last, first or in between."""
    M, past, D = 9, 1500, 64
    masks, _ = ql.tree_masks(tree(M, 5))
    at = np.arange(past + M)
    for line in (at / 60, at / 5, (past - at) / 60, np.where(at % 200 == 199, at / 20, 0), 12 * np.sin(at / 40)):
        def edit(c):
            c.q[:, :, 0] = 4
            c.k[:, :, 0] = (line * 2).astype(c.k.dtype)[:, None]             # score 1 line
        run(ql, ctx, M, 4, 2, D, past, half, masks, 20, edit=edit)


def test_equal_scores(ql, ctx):
    """A query of zeros: the mean of what is seen, over a long context."""
    for half in (False, True):
        def edit(c):
            c.q[:] = 0
        run(ql, ctx, 2, 4, 1, 64, 5000, half, ql.tree_masks([-1, -1])[0], 19, edit=edit)


def test_cache_offsets_past_32_bits(ql, ctx):
    """A half cache of 4.5 GiB a region: its last keys."""
    M, H, KV, D = 4, 16, 16, 256
    row = KV * D * 2
    T = (9 << 29) // row
    g = np.random.default_rng(1)
    act = Box(ql, ctx)
    q = (0.3 * g.standard_normal((M, H, D))).astype(np.float32)
    masks, _ = ql.tree_masks([-1, 0, 0, 2])
    act.put("q", q)
    act.put("mask", masks)
    act.put("out", np.zeros((M, H, D), np.float32))
    act.place()
    cache = ctx.arena(2 * T * row)
    # keys of -60000 along one direction vanish from the softmax; only the last 100 and the drafted rows count
    zeros = np.zeros((1 << 14, KV, D), np.float16)
    zeros[:, :, 0] = -60000
    q[:, :, 0] = 50.0
    act.arena.write(act.off("q"), q)
    blank = np.zeros_like(zeros)
    for s in range(0, T, 1 << 14):
        n = min(1 << 14, T - s)
        cache.write(s * row, zeros[:n])
        cache.write((T + s) * row, blank[:n])
    tail = 100 + M
    k, v = (g.standard_normal((tail, KV, D)).astype(np.float16) for _ in range(2))
    cache.write((T - tail) * row, k)
    cache.write((2 * T - tail) * row, v)
    ctx.attention_tree(act.arena, act.off("q"), cache, 0, T * row, ql.DTYPE_F16, T, M, H, KV, D, T - M, act.off("mask"), act.off("out"))
    want, tol = formula(q, k, v, seen_of(masks, M, 100))
    got = act.get("out")
    assert (np.abs(got - want) <= tol + 2 * np.sqrt(T) * U).all()
    act.release()
    cache.release()


def test_same_bits_every_time(ql, ctx):
    for M, past, half in ((3, 5000, False), (40, 900, True)):
        c = Call(ql, ctx, M, 28, 4, 128, past, half, ql.tree_masks(tree(M, 1))[0], 20)
        ctx.attention_tree(*c.args)
        a = c.out().copy()
        for _ in range(4):
            ctx.attention_tree(*c.args)
        assert np.array_equal(c.out().view(np.uint32), a.view(np.uint32))
        c.release()


def test_graph_on_another_context(ql):
    """Captured on one context, replayed on another beside the first one's own calls (each has its workspace), and after it."""
    a, b = ql.Context(0), ql.Context(0)
    one = Call(ql, b, 6, 28, 4, 128, 3000, False, ql.tree_masks(tree(6, 1))[0], 21)
    two = Call(ql, b, 9, 28, 4, 128, 2500, True, ql.tree_masks(tree(9, 2))[0], 22)
    for c in (one, two):
        b.attention_tree(*c.args)
    b.sync()
    want = [c.out().copy() for c in (one, two)]
    a.graph_begin()
    a.attention_tree(*one.args)
    g = a.graph_end()
    a._owned.discard(g)
    for _ in range(5):
        for c in (one, two):
            c.act.arena.write(c.act.off("out"), np.zeros((c.dims[0] * c.dims[1], c.dims[3]), np.float32))
        ql._check(ql.lib().ql_graph_launch(b.handle, g.handle))
        a.attention_tree(*two.args)
        a.sync()
        b.sync()
        assert np.array_equal(one.out(), want[0]) and np.array_equal(two.out(), want[1])
    a.destroy()
    one.act.arena.write(one.act.off("out"), np.zeros((6 * 28, 128), np.float32))
    ql._check(ql.lib().ql_graph_launch(b.handle, g.handle))
    b.sync()
    assert np.array_equal(one.out(), want[0])
    ql._check(ql.lib().ql_graph_destroy(g.handle))
    g.handle = None
    one.release()
    two.release()
    b.destroy()


def test_refusals(ql, ctx):
    M, H, KV, D, past = 4, 4, 2, 32, 10
    c = Call(ql, ctx, M, H, KV, D, past, False, ql.tree_masks([-1, 0, 0, 1])[0], 1)
    a, size, csize = list(c.args), c.act.arena.size, c.cache.arena.size

    def refused(name, **at):
        b = list(a)
        for i, v in at.items():
            b[int(i[1:])] = v
        with pytest.raises(ql.QlError) as e:
            ctx.attention_tree(*b)
        assert e.value.name == name, (at, e.value)

    for at in ({"_7": 0}, {"_7": 257}, {"_8": 3}, {"_8": 0}, {"_9": 0}, {"_10": 4}, {"_10": 12}, {"_10": 264}, {"_11": -1}, {"_5": 2}, {"_6": 0}):
        refused("QL_E_INVALID", **at)
    for at in ({"_6": past + M - 1}, {"_11": 1 << 30}, {"_1": size}, {"_13": size - 16}, {"_12": size}, {"_3": csize - 64}, {"_4": csize}, {"_6": 1 << 20}):
        refused("QL_E_RANGE", **at)
    for at in ({"_1": a[1] + 8}, {"_13": a[13] + 4}, {"_3": a[3] + 8}, {"_4": a[4] + 4}, {"_12": a[12] + 4}):
        refused("QL_E_ALIGN", **at)
    for at in ({"_13": a[1]}, {"_13": a[1] + 16}, {"_13": a[12] // 16 * 16}, {"_0": a[2], "_1": a[4], "_12": None, "_13": a[3]}):
        refused("QL_E_INVALID", **at)
    ctx.attention_tree(*a)
    c.check()
    c.release()


def test_refuses_more_keys_than_it_counts(ql, ctx):
    c = Call(ql, ctx, 4, 4, 2, 32, 10, False, None, 1)
    a = list(c.args)
    a[6] = (1 << 31) - 1
    for past in ((1 << 30) + 1, (1 << 31) - 8):
        a[11] = past
        with pytest.raises(ql.QlError) as e:
            ctx.attention_tree(*a)
        assert e.value.name == "QL_E_INVALID"
    c.release()


def many(q, k, v, seen):
    """formula()'s results for a head's rows at once."""
    M, H, D = q.shape
    T, KV, _ = k.shape
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    out, tol = np.zeros((M, H, D)), np.zeros((M, H, D))
    with np.errstate(all="ignore"):
        for h in range(H):
            kh, vh = k[:, h // (H // KV)], v[:, h // (H // KV)]
            score = np.where(seen, q[:, h] @ kh.T / np.sqrt(D), -np.inf)
            p = np.exp(score - score.max(1, keepdims=True))
            total = p.sum(1, keepdims=True)
            fine = np.isfinite(vh)
            o = p @ np.where(fine, vh, 0)
            for key, d in np.argwhere(~fine):
                o[:, d] += np.where(seen[:, key], p[:, key] * vh[key, d], 0)
            a = np.where(seen, np.abs(q[:, h]) @ np.where(np.isfinite(kh), np.abs(kh), 0).T, 0).max(1, keepdims=True) / np.sqrt(D)
            bad = (np.isnan(score) | (score == np.inf)).any(1)
            any_seen = seen.any(1)
            out[:, h] = np.where(any_seen[:, None], np.where(bad[:, None], np.nan, o / total), 0)
            tol[:, h] = np.where(any_seen[:, None], (32 * a + 32 + 2 * np.sqrt(T)) * U * (p @ np.where(fine, np.abs(vh), 0)) / total, 0)
    return out, tol


def run_many(ql, ctx, M, H, KV, D, past, half, masks, seed, **kw):
    c = Call(ql, ctx, M, H, KV, D, past, half, masks, seed, **kw)
    ctx.attention_tree(*c.args)
    c.check(many(c.q, c.k, c.v, seen_of(masks, M, past)))
    c.release()


# Shapes of the instances with 32 pairs a workgroup, and of more than 64 key ranges, whose merge has two weights a lane.
PLANS = [
    # M, H, KV, D, past, half, (pairs, waves, key ranges), label
    (251, 5, 1, 64, 40, False, (32, 4, 3), "1255 pairs of a kv head, a last group of 7"),
    (140, 9, 1, 128, 33, False, (32, 4, 2), "heads of 128, a last group of 12"),
    (25, 28, 4, 128, 3980, False, (32, 4, 16), "a tree after a long context, a last group of 15"),
    (65, 33, 1, 64, 1950, True, (32, 4, 1), "a half cache, a last group of 1"),
    (129, 17, 1, 128, 2000, True, (32, 4, 1), "a half cache, heads of 128, a last group of 17"),
    (40, 40, 1, 64, 3200, True, (32, 4, 7), "a half cache, ranges that are merged"),
    (1, 28, 4, 128, 20000, False, (16, 4, 79), "more than 64 key ranges"),
    (1, 28, 4, 128, 20000, True, (16, 4, 79), "more than 64 key ranges of a half cache"),
    (3, 6, 2, 200, 32700, True, (16, 4, 128), "as many key ranges as there are"),
]


@pytest.mark.parametrize("M,H,KV,D,past,half,plan,label", PLANS)
def test_planned_instances(ql, ctx, M, H, KV, D, past, half, plan, label):
    print(label, flush=True)
    info = ql.plan_attention_tree(ql.DTYPE_F16 if half else ql.DTYPE_F32, past + M, M, H, KV, D, past)
    assert (info.pairs, info.waves, info.nsplit) == plan
    c = Call(ql, ctx, M, H, KV, D, past, half, ql.tree_masks(tree(M, M))[0], past)
    ctx.attention_tree(*c.args)
    first = c.check(many(c.q, c.k, c.v, seen_of(c.masks, M, past)))
    for _ in range(3):
        ctx.attention_tree(*c.args)
    assert np.array_equal(c.out(), first.astype(np.float32))
    c.release()


WIDE = [p[:6] for p in PLANS if p[6][0] == 32 and p[4] < 3000]


@pytest.mark.parametrize("M,H,KV,D,past,half", WIDE)
def test_32_pairs_without_a_mask(ql, ctx, M, H, KV, D, past, half):
    """Causal rows: with the chain's mask the bits are the same."""
    c = Call(ql, ctx, M, H, KV, D, past, half, None, M)
    ctx.attention_tree(*c.args)
    got = c.check(many(c.q, c.k, c.v, seen_of(None, M, past)))
    d = Call(ql, ctx, M, H, KV, D, past, half, ql.tree_masks(np.arange(-1, M - 1))[0], M)
    ctx.attention_tree(*d.args)
    assert np.array_equal(d.out(), got)
    c.release()
    d.release()


@pytest.mark.parametrize("M,H,KV,D,past,half", WIDE)
@pytest.mark.parametrize("what,value", [("k", np.nan), ("v", np.inf), ("k", -np.inf)])
def test_32_pairs_of_what_is_not_finite(ql, ctx, M, H, KV, D, past, half, what, value):
    """In a drafted row that a few see, and (a second call) in the context: on the VALU again, both tiles of a wave. Some rows see
    nothing of the tree."""
    masks, _ = ql.tree_masks(tree(M, 3))
    masks[[0, M // 2]] = 0
    for key in (past + 2 * M // 3, past // 2):
        def edit(c):
            getattr(c, what)[key, :, 5] = value
        run_many(ql, ctx, M, H, KV, D, past, half, masks, 11, edit=edit)


@pytest.mark.parametrize("M,H,KV,D,half", [(256, 5, 1, 64, False), (128, 9, 1, 128, False), (256, 64, 1, 64, True), (256, 64, 1, 128, True)])
def test_32_pairs_that_see_nothing(ql, ctx, M, H, KV, D, half):
    """No context, masks of any bits and of none: rows of zeros among the others, whole workgroups of them at the end."""
    assert ql.plan_attention_tree(ql.DTYPE_F16 if half else ql.DTYPE_F32, M, M, H, KV, D, 0).pairs == 32
    g = np.random.default_rng(M)
    masks = g.integers(0, 2**63, (M, M // 64)).astype(np.uint64)
    masks[::7] = 0
    masks[M - 40:] = 0
    run_many(ql, ctx, M, H, KV, D, 0, half, masks, 5)


@pytest.mark.parametrize("M,H,KV,D,past,half", WIDE)
def test_32_pairs_with_scores_that_rise(ql, ctx, M, H, KV, D, past, half):
    """Along the context, slowly and by leaps, for one tile of a wave and not for the other."""
    masks, _ = ql.tree_masks(tree(M, 5))
    at = np.arange(past + M)
    for line in (at / 40, np.where(at % 90 == 89, at / 9, 0), (past - at) / 40):
        def edit(c):
            c.q[:, :, 0] = np.where(np.arange(M)[:, None] % 5 == 0, 4, 0.01)
            c.k[:, :, 0] = (line * 2).astype(c.k.dtype)[:, None]
        run_many(ql, ctx, M, H, KV, D, past, half, masks, 20, edit=edit)


@pytest.mark.parametrize("past,low", [(40000, 20), (300000, 22), (300000, 24)])
def test_long_tails_of_small_weights(ql, ctx, past, low):
    """One key far above all the others over a long half cache: V is 0 at the key and 1 elsewhere, so the result is the others' part,
    t / (1 + t) with t = (T - 1) e^-low. Its relative error: the scores' 16 u A twice, A = low, and the sums' (32 + 2 sqrt(T)) u. A weight's
    two parts end at half a step of 2^-24 of 2^8 of it: 2^-33 of the reference, which T weights lose at most T times."""
    M, H, KV, D = 2, 2, 1, 64
    g = np.random.default_rng(past)
    act, cache = Box(ql, ctx), Box(ql, ctx)
    T = past + M
    q = np.zeros((M, H, D), np.float32)
    q[:, :, 0] = low * 8                                                     # sqrt(D): a key's first value times `low` is its score
    k, v = np.zeros((T, KV, D), np.float16), np.ones((T, KV, D), np.float16)
    at = int(g.integers(past))
    k[at, :, 0], v[at] = 1, 0
    act.put("q", q)
    act.put("out", np.zeros((M, H, D), np.float32))
    cache.put("k", k)
    cache.put("v", v)
    act.place()
    cache.place()
    ctx.attention_tree(act.arena, act.off("q"), cache.arena, cache.off("k"), cache.off("v"), ql.DTYPE_F16, T, M, H, KV, D, past, None, act.off("out"))
    for m, row in enumerate(act.get("out").astype(np.float64)):
        t = (past + m // H) * np.exp(-np.float64(low))
        want = t / (1 + t)
        assert np.abs(row - want).max() <= (32 * low + 32 + 2 * np.sqrt(T)) * U * want + T * 2.0 ** -33
    act.release()
    cache.release()
