"""GPU: log probabilities, entropy and top alternatives (ql_token_logprobs) against 64-bit sums over the same fp32 logits.

Rounding, in units u = 2^-24: ln S of a sum of positive terms is off by the exponentials' own error (2 u and |x - m| u for the
rounded difference, weighted by the terms: at most 2 + H + 1 of them, H the entropy plus ln V at most 17) and by the additions,
which the kernel makes in runs of at most some tens and then pairwise: 64 u. x - m and the last subtraction add 2 |log p| u:
(100 + 3 |log p|) u. The entropy's second sum has its terms' relative error besides: (200 + 3 H + 100 H) u."""
import numpy as np
import pytest

from tests.arena_box import Box

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, tokens, top):
    M, V = x.shape
    lp64, ent = np.empty((M, V)), np.empty(M)
    for m in range(M):
        r = x[m].astype(np.float64)
        if np.isnan(r).any() or (r == np.inf).any():
            lp64[m], ent[m] = np.nan, np.nan
            continue
        mx = r.max()
        if mx == -np.inf:
            lp64[m], ent[m] = -np.inf, 0
            continue
        e = np.exp(r - mx)
        lp64[m] = r - mx - np.log(e.sum())
        p = e / e.sum()
        ent[m] = -(p[p > 0] * lp64[m][p > 0]).sum()
    lp = np.zeros(tokens.shape)
    for m, t in np.ndindex(tokens.shape):
        if 0 <= tokens[m, t] < V:
            lp[m, t] = lp64[m, tokens[m, t]]
    ids, tlp = np.full((M, top), -1, np.int32), np.full((M, top), -np.inf)
    for m in range(M):
        key = np.where(np.isnan(x[m]), np.inf, x[m]).astype(np.float64)
        order = np.lexsort((np.arange(V), -key, ~np.isnan(x[m])))[:top]
        ids[m, :len(order)], tlp[m, :len(order)] = order, lp64[m, order]
    return lp, ent, ids, tlp


class Call:
    def __init__(self, ql, ctx, x, tokens, top, stride=None, gap=0, entropy=True):
        M, V = x.shape
        self.M, self.top = M, top
        stride = V if stride is None else stride
        full = np.full((M, stride), 1e30, np.float32)
        full[:, :V] = x
        self.box = b = Box(ql, ctx)
        b.put("x", full.reshape(-1)[:(M - 1) * stride + V], gap=gap)
        b.put("tok", tokens.astype(np.int32), gap=gap)
        for n, a in (("lp", np.full(tokens.size + 3, 5, np.float32)), ("ent", np.full(M + 3, 5, np.float32)),
                     ("ids", np.full(M * top + 3, 5, np.int32)), ("tlp", np.full(M * top + 3, 5, np.float32))):
            b.put(n, a, gap=gap)
        b.place()
        self.shape = tokens.shape
        self.args = (b.arena, b.off("x"), stride, M, V, b.off("tok"), tokens.shape[1], top, b.off("lp"), b.off("ent") if entropy else None,
                     b.off("ids"), b.off("tlp"))
        self.entropy = entropy

    def results(self):
        b, n, k = self.box, self.shape[0] * self.shape[1], self.M * self.top
        out = [b.get("lp"), b.get("ent"), b.get("ids"), b.get("tlp")]
        for a, size in zip(out, (n, self.M if self.entropy else 0, k, k)):
            assert (a[size:] == 5).all()                                     # what lies behind stays
        return out[0][:n].reshape(self.shape), out[1][:self.M], out[2][:k].reshape(self.M, self.top), out[3][:k].reshape(self.M, self.top)


def close(got, want, tol):
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)].astype(np.float32))
    if fine.any():
        off = np.abs(got[fine].astype(np.float64) - want[fine]) - tol[fine]
        assert off.max() <= 0, off.max()


def compare(call, x, tokens, top):
    lp, ent, ids, tlp = call.results()
    rlp, rent, rids, rtlp = reference(x, tokens, top)
    close(lp, rlp, (100 + 3 * np.abs(rlp)) * U)
    if call.entropy:
        close(ent, rent, (200 + 103 * np.abs(rent)) * U)
    assert np.array_equal(ids, rids)
    close(tlp, rtlp, (100 + 3 * np.abs(rtlp)) * U)


def run(ql, ctx, x, tokens, top, **kw):
    c = Call(ql, ctx, x, tokens, top, **kw)
    ctx.token_logprobs(*c.args)
    compare(c, x, tokens, top)
    c.box.release()


@pytest.mark.parametrize("M,V,T,top", [
    (1, 1, 1, 1), (2, 2, 1, 5), (1, 3, 2, 32), (3, 31, 4, 32), (5, 64, 0, 1), (2, 255, 3, 20), (2, 256, 1, 32), (3, 257, 1, 32), (4, 1000, 256, 7),
    (2, 4095, 1, 32), (2, 4096, 2, 20), (2, 4097, 1, 32), (7, 8191, 1, 5), (3, 8193, 1, 32), (2, 20000, 1, 31), (1, 151936, 1, 20), (5, 151936, 4, 32), (2, 151937, 1, 32),
    (33, 12345, 1, 0), (300, 777, 2, 3), (1, 1000003, 1, 32)])
def test_matches_sums_in_64_bits(ql, ctx, M, V, T, top):
    g = np.random.default_rng(V + M)
    x = (3 * g.standard_normal((M, V))).astype(np.float32)
    tokens = g.integers(-1, V, (M, T))
    run(ql, ctx, x, tokens, top)


@pytest.mark.parametrize("stride,gap", [(1001, 4), (1004, 8), (1000, 12), (4000, 0)])
def test_strides_and_alignment(ql, ctx, stride, gap):
    """Rows apart, offsets of any multiple of 4; what lies between rows is not read (1e30)."""
    g = np.random.default_rng(stride)
    x = (2 * g.standard_normal((6, 1000))).astype(np.float32)
    run(ql, ctx, x, g.integers(0, 1000, (6, 2)), 32, stride=stride, gap=gap)


def test_equal_logits_go_to_the_lower_id(ql, ctx):
    for V in (40, 700, 5000, 151936):
        x = np.zeros((4, V), np.float32)
        x[1, ::3] = 1.0
        x[2] = np.where(np.arange(V) % 2, 0.0, -0.0)                          # equal, whatever the sign
        x[3, -20:] = 2.0
        run(ql, ctx, x, np.zeros((4, 1), np.int64), 32)
    # in descending and ascending order: the best are all in one place
    x = np.stack([np.arange(20000), -np.arange(20000)]).astype(np.float32) * 0.01
    run(ql, ctx, x, np.zeros((2, 1), np.int64), 32)


def test_masks_and_extremes(ql, ctx):
    V, low = 3000, np.finfo(np.float32).min
    g = np.random.default_rng(5)
    x = g.standard_normal((12, V)).astype(np.float32)
    x[0] = -np.inf                                                           # nothing allowed
    x[1] = -np.inf
    x[1, 2999] = 3.0                                                         # one token
    x[2, 5:] = -np.inf                                                       # fewer than asked for
    x[3] = low                                                               # the type's lowest value everywhere
    x[4] = low
    x[4, 77] = 0
    x[5] = 1e30 * x[5]                                                       # far apart
    x[6] += 1e6                                                              # large
    x[7, 100] = np.nan
    x[8, [5, 200]] = -np.nan
    x[9, 30] = np.inf
    x[10] *= 1e-40                                                           # subnormal
    x[11, :] = np.finfo(np.float32).max
    run(ql, ctx, x, np.tile(np.array([[77, 2999, -1, V, 2**31 - 1, 100]]), (12, 1)), 32)
    # a row of another wave's, chunk's size: the mask leaves the last element alone
    y = np.full((3, 70001), -np.inf, np.float32)
    y[1, 70000] = 1
    y[2, [1, 40000, 70000]] = [1, 1, 2]
    run(ql, ctx, y, np.array([[0], [70000], [40000]]), 5)


def test_only_what_is_asked_for(ql, ctx):
    g = np.random.default_rng(6)
    x = g.standard_normal((3, 500)).astype(np.float32)
    run(ql, ctx, x, g.integers(0, 500, (3, 2)), 0, entropy=False)
    run(ql, ctx, x, np.zeros((3, 0), np.int64), 4, entropy=False)
    run(ql, ctx, x, np.zeros((3, 0), np.int64), 0)


def test_same_bits_every_time(ql, ctx):
    g = np.random.default_rng(8)
    x = (3 * g.standard_normal((9, 60001))).astype(np.float32)
    c = Call(ql, ctx, x, g.integers(0, 60001, (9, 3)), 20)
    ctx.token_logprobs(*c.args)
    first = [a.copy() for a in c.results()]
    for _ in range(5):
        ctx.token_logprobs(*c.args)
    for a, b in zip(first, c.results()):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    c.box.release()


def test_graph_replays(ql, ctx):
    """Captured once, replayed on other logits between the context's own calls."""
    g = np.random.default_rng(9)
    c = Call(ql, ctx, (3 * g.standard_normal((4, 30000))).astype(np.float32), g.integers(0, 30000, (4, 2)), 20)
    other = Call(ql, ctx, (3 * g.standard_normal((7, 50001))).astype(np.float32), g.integers(0, 50001, (7, 2)), 20)
    ctx.graph_begin()
    ctx.token_logprobs(*c.args)
    graph = ctx.graph_end()
    tokens = c.box.items["tok"][1]
    for i in range(4):
        x = (3 * g.standard_normal((4, 30000))).astype(np.float32)
        c.box.arena.write(c.box.off("x"), x)
        ctx.token_logprobs(*other.args)
        graph.launch()
        ctx.token_logprobs(*other.args)
        ctx.sync()
        compare(c, x, tokens, 20)
        compare(other, other.box.items["x"][1].reshape(7, -1), other.box.items["tok"][1], 20)
    graph.destroy()
    c.box.release()
    other.box.release()


def test_more_rows_than_a_workspace_holds(ql, ctx):
    """65535 rows."""
    g = np.random.default_rng(10)
    M, V = 65535, 301
    x = (2 * g.standard_normal((M, V))).astype(np.float32)
    tokens = g.integers(0, V, (M, 1))
    c = Call(ql, ctx, x, tokens, 2)
    ctx.token_logprobs(*c.args)
    lp, ent, ids, tlp = c.results()
    r = x.astype(np.float64)
    mx = r.max(1, keepdims=True)
    full = r - mx - np.log(np.exp(r - mx).sum(1, keepdims=True))
    want = np.take_along_axis(full, tokens, 1)
    assert (np.abs(lp - want) <= (100 + 3 * np.abs(want)) * U).all()
    H = -(np.exp(full) * full).sum(1)
    assert (np.abs(ent - H) <= (200 + 103 * H) * U).all()
    order = np.argsort(-x, axis=1, kind="stable")[:, :2]
    assert np.array_equal(ids, order)
    want = np.take_along_axis(full, order, 1)
    assert (np.abs(tlp - want) <= (100 + 3 * np.abs(want)) * U).all()
    c.box.release()


def test_refusals(ql, ctx):
    g = np.random.default_rng(1)
    c = Call(ql, ctx, g.standard_normal((4, 100)).astype(np.float32), g.integers(0, 100, (4, 2)), 3)
    a, size = list(c.args), c.box.arena.size

    def refused(name, **at):
        b = list(a)
        for i, v in at.items():
            b[int(i[1:])] = v
        with pytest.raises(ql.QlError) as e:
            ctx.token_logprobs(*b)
        assert e.value.name == name, (at, e.value)

    for at in ({"_3": 0}, {"_3": 65536}, {"_6": -1}, {"_6": 257}, {"_7": -1}, {"_7": 33}, {"_6": 0, "_7": 0, "_9": None}):
        refused("QL_E_INVALID", **at)
    for at in ({"_4": 0}, {"_2": 99}, {"_4": (1 << 24) + 1, "_2": (1 << 24) + 1}):
        refused("QL_E_DIMS", **at)
    for at in ({"_1": size}, {"_5": size - 4}, {"_8": size}, {"_9": size}, {"_10": size}, {"_11": size}, {"_2": 1 << 20}):
        refused("QL_E_RANGE", **at)
    for i in (1, 5, 8, 9, 10, 11):
        refused("QL_E_ALIGN", **{f"_{i}": a[i] + 2})
    for at in ({"_8": a[1]}, {"_9": a[1] + 1596}, {"_10": a[5]}, {"_11": a[10]}, {"_9": a[8]}):
        refused("QL_E_INVALID", **at)
    ctx.token_logprobs(*a)
    c.box.release()


@pytest.mark.parametrize("V", [16384, 70000, 151936, 262145, 600001])
def test_few_alternatives(ql, ctx, V):
    """Numbers of alternatives about the one at which the parts' largest are joined at once, over few and many parts."""
    g = np.random.default_rng(V)
    x = (3 * g.standard_normal((2, V))).astype(np.float32)
    x[1, g.integers(0, V, 40)] = 20.0                                        # equal ones in many parts
    for top in (1, 3, 4, 5, 6, 7, 8, 12, 13):
        run(ql, ctx, x, g.integers(0, V, (2, 1)), top)


def sure(x):
    """(log probabilities [V], entropy) of a row with few logits far above the others: the rest's terms R are summed apart from the n
    largest ones, so that 64 bits hold ln S = ln n + ln(1 + R / n) to 2^-50 of itself."""
    d = x.astype(np.float64) - x.max()
    rest = d < 0
    n, R = (~rest).sum(), np.exp(d[rest]).sum()
    ls = np.log(n) + np.log1p(R / n)
    return d - ls, ls - (d[rest] * np.exp(d[rest])).sum() / (n + R)


@pytest.mark.parametrize("gap", [3, 8, 12, 17, 24, 30])
@pytest.mark.parametrize("V", [2, 50, 1001, 30000, 151936])
def test_sure_rows(ql, ctx, V, gap):
    """One logit far above the others, or several alike: a log probability and an entropy far below 1, to their own rounding.
    A term e^d is off by (2.3 |d| + 4) u (the difference's rounding, log2 e's and the product's, two exponentials), d at most gap + 6 here;
    R's additions and the product with d by some 50 u: (2.3 (gap + 6) + 54) u of ln S and of the entropy, and one rounding."""
    g = np.random.default_rng(V + gap)
    x = np.zeros((6, V), np.float32)
    x[:3] = np.clip(g.standard_normal((3, V)), -3, 3)
    at = [V // 2, 0, V - 1, V // 3, 0, V - 1]
    for m in range(6):
        x[m, at[m]] = x[m].max() + gap if m < 3 else gap
    x[4, V - 1] = gap                                                        # two alike, far apart
    x[5, ::7] = gap                                                          # many alike
    tokens = np.stack([at, [(a + 1) % V for a in at]], 1)
    top = min(V, 3)
    c = Call(ql, ctx, x, tokens, top)
    ctx.token_logprobs(*c.args)
    lp, ent, ids, tlp = (a.astype(np.float64) for a in c.results())
    for m in range(6):
        want, H = sure(x[m])
        r = (2.3 * (gap + 6) + 56) * U
        ls = -want.max()
        assert abs(ent[m] - H) <= r * H, (m, ent[m], H)
        assert (np.abs(lp[m] - want[tokens[m]]) <= r * ls + U * np.abs(want[tokens[m]])).all()
        order = np.argsort(-x[m], kind="stable")[:top]
        assert np.array_equal(ids[m], order)
        assert (np.abs(tlp[m] - want[order]) <= r * ls + U * np.abs(want[order])).all()
    c.box.release()


def test_rows_that_pass_through_the_workspace_in_turn(ql, ctx):
    """More rows than 64 MiB of partial sums hold at once: 48 bytes per 1024 logits, 9383 rows of 151936. 97 different rows take turns,
    so that a row's place shows in its results on both sides of the border."""
    g = np.random.default_rng(12)
    V, M, N = 151936, 9383 + 20, 97
    assert (64 << 20) // (48 * -(-V // 1024)) == M - 20
    x = (2 * g.standard_normal((N, V))).astype(np.float32)
    x[5] = -np.inf
    x[7, 3] = np.nan
    tokens = g.integers(-1, V, (N, 2))
    lp, ent, ids, tlp = reference(x, tokens, 3)
    lay, size = ql.ArenaLayout(), 4 * V * M
    off = {n: lay.take(b) for n, b in (("x", size), ("tok", 8 * M), ("lp", 8 * M + 64), ("ent", 4 * M + 64), ("ids", 12 * M + 64), ("tlp", 12 * M + 64))}
    arena = ctx.arena(lay.used)
    for m in range(0, M, N):
        n = min(N, M - m)
        arena.write(off["x"] + 4 * V * m, x[:n])
    at = np.arange(M) % N
    arena.write(off["tok"], tokens[at].astype(np.int32))
    for n in ("lp", "ent", "ids", "tlp"):
        arena.write(off[n], np.full(3 * M + 16 if n in ("ids", "tlp") else 2 * M + 16 if n == "lp" else M + 16, 5, np.float32))
    ctx.token_logprobs(arena, off["x"], V, M, V, off["tok"], 2, 3, off["lp"], off["ent"], off["ids"], off["tlp"])
    close(arena.read(off["lp"], (M, 2), np.float32), lp[at], ((100 + 3 * np.abs(lp)) * U)[at])
    close(arena.read(off["ent"], (M,), np.float32), ent[at], ((200 + 103 * np.abs(ent)) * U)[at])
    assert np.array_equal(arena.read(off["ids"], (M, 3), np.int32), ids[at])
    close(arena.read(off["tlp"], (M, 3), np.float32), tlp[at], ((100 + 3 * np.abs(tlp)) * U)[at])
    for n, size in (("lp", 8 * M), ("ent", 4 * M), ("ids", 12 * M), ("tlp", 12 * M)):
        assert (arena.read(off[n] + size, (16,), np.float32) == 5).all()
    arena.release()
