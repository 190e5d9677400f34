"""ql_paged_attention against 64-bit arithmetic: decoding rows, pieces and whole prompts in one batch, fp16 and e4m3 pages, fp32 and fp16
rows, contexts from one token on, poisoned memory where nothing may be seen, tables that say what they may not."""
import numpy as np
import pytest

from tests.arena_box import Box
from tests.paged_ref import Batch, Cache, attention, f8_encode

pytestmark = pytest.mark.gpu

DECODE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 300)]
MIXED = [(1, 700), (70, 70), (0, 5), (33, 500), (1, 3), (5, 64), (200, 200), (2, 1500)]

CASES = [  # seqs, page, H, KV, D
    (DECODE, 64, 14, 2, 64),
    (DECODE, 256, 28, 4, 128),
    ([(1, 5000)], 128, 28, 4, 128),
    ([(1, 1000 + 37 * i) for i in range(20)], 64, 14, 2, 64),
    ([(1, 40)] * 130, 64, 4, 4, 64),
    (MIXED, 64, 14, 2, 64),
    (MIXED, 128, 28, 4, 128),
    (MIXED, 64, 6, 3, 96),
    ([(1, 90), (3, 130), (40, 64)], 64, 40, 1, 80),
    ([(1, 90), (3, 130), (40, 200)], 64, 5, 5, 256),
    ([(1, 90), (17, 33)], 64, 64, 2, 16),
    ([(400, 400), (300, 1000)], 64, 16, 16, 128),
    ([(1, 70), (90, 170)], 64, 12, 2, 192),
    ([(1, 30)] * 50 + [(50, 700), (33, 33), (0, 4)] * 7, 64, 8, 2, 64),         # more sequences than a wave has lanes, of both kinds
    ([(40, 2000)], 128, 9, 3, 64),                                               # parts of a tile's tokens, kv heads that do not divide 512
    ([(1, 1100), (20, 1200)], 64, 96, 1, 32),                                    # a row of more pairs than the few have
    ([(500, 500), (1, 9), (300, 900)], 64, 64, 4, 64),                           # many rows: tiles of 128 pairs, and below of each kind of D
    ([(600, 600), (200, 700), (1, 1)], 128, 64, 8, 128),
    ([(790, 800)], 64, 64, 8, 96),
    ([(790, 790)], 64, 64, 2, 32),
    ([(1, 1500 + 9 * i) for i in range(40)] + [(30, 2000)], 64, 16, 4, 64),      # whole tiles of many sequences beside one of many rows
]


class Call:
    def __init__(self, ql, ctx, batch, H, KV, D, f8, q16, seed=1, cache=None, q=None, spread=2.0, **desc):
        g = np.random.default_rng(seed)
        self.ql, self.ctx, self.batch, self.H, self.q16 = ql, ctx, batch, H, q16
        self.cache = cache or Cache(f8, batch.n_page, batch.page, KV, D, seed)
        t = np.float16 if q16 else np.float32
        self.q = (spread * g.standard_normal((batch.M, H, D))).astype(t) if q is None else q.astype(t)
        self.before = g.standard_normal((batch.M, H, D)).astype(t)
        self.box = box = Box(ql, ctx)
        box.put("q", self.q), box.put("out", self.before)
        batch.put(box), self.cache.put(box)
        box.place()
        self.paged, self.desc = self.cache.desc(ql, box), batch.desc(ql, box, **desc)

    @property
    def dtype(self):
        return self.ql.DTYPE_F16 if self.q16 else self.ql.DTYPE_F32

    def run(self, ctx=None, sync=True):
        box, c = self.box, ctx or self.ctx
        c.paged_attention(box.arena, box.off("q"), self.dtype, box.arena, self.paged, self.desc, self.batch.M, self.H, box.off("out"))
        if sync:
            c.sync()

    def want(self):
        out, tol, size = attention(self.q, self.cache, self.batch)
        # fp16: each probability and the result are rounded once, the result's own range ends at 2^-25
        return out, tol + (2.0 ** -11 * (size + np.abs(out)) + 2.0 ** -25 if self.q16 else 0)

    def check(self, skip=(), want=None):
        out, tol = want or self.want()
        got = self.box.get("out")
        b = self.batch
        there = np.zeros(b.M, bool)
        for s, (n, _) in enumerate(b.seqs):
            there[b.row_start[s]:b.row_start[s] + n] = s not in skip
        out, tol, now = out[there], tol[there], got[there].astype(np.float64)
        odd = ~np.isfinite(out)
        assert np.array_equal(np.isnan(now), np.isnan(out))
        assert np.array_equal(now[odd & ~np.isnan(out)], out[odd & ~np.isnan(out)])
        worst = np.max(np.abs(now[~odd] - out[~odd]) / tol[~odd], initial=0)
        assert worst <= 1, worst
        assert np.array_equal(got[~there].view(np.uint8), self.before[~there].view(np.uint8))
        return got


@pytest.mark.parametrize("q16", [False, True])
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(ql, ctx, case, f8, q16):
    seqs, page, H, KV, D = CASES[case]
    call = Call(ql, ctx, Batch(seqs, page, seed=case, pad=2), H, KV, D, f8, q16, seed=case)
    call.run()
    first = call.check()
    call.run()                                                                   # the same bits again
    assert np.array_equal(call.box.get("out").view(np.uint8), first.view(np.uint8))
    call.box.release()


@pytest.mark.parametrize("q16", [False, True])
@pytest.mark.parametrize("f8", [False, True])
def test_what_no_row_sees(ql, ctx, f8, q16):
    """Memory behind the sequences' ends, and the scales of groups without tokens, hold NaN; so do spare pages."""
    batch = Batch([(1, 33), (20, 50), (1, 129), (90, 90), (1, 1), (64, 64)], 64, seed=3)
    full = Cache(f8, batch.n_page, 64, 2, 64, 9)
    cache = Cache(f8, batch.n_page, 64, 2, 64, 9, empty=True)
    used = np.concatenate([batch.places(s) for s in range(len(batch.seqs))])
    for n in "kv":
        a, b = getattr(cache, n).reshape(-1, 2, 64), getattr(full, n).reshape(-1, 2, 64)
        a[used] = b[used]
        if f8:
            cache.scale[n].reshape(-1, 2)[used // 16] = full.scale[n].reshape(-1, 2)[used // 16]
    call = Call(ql, ctx, batch, 6, 2, 64, f8, q16, cache=cache)
    call.run()
    call.check()
    call.box.release()


@pytest.mark.parametrize("seqs", [[(70, 70)], [(70, 600)], [(2, 200), (150, 150)], [(3, 3)]])
@pytest.mark.parametrize("f8", [False, True])
def test_tokens_that_are_not_finite(ql, ctx, f8, seqs):
    """A later token's key or value of infinities and NaN changes no earlier row; the rows that see it have the formula's."""
    batch = Batch(seqs, 64, seed=5)
    cache = Cache(f8, batch.n_page, 64, 2, 64, 6)
    for s, (n, L) in enumerate(seqs):
        at = batch.places(s)
        v, k = cache.v.reshape(-1, 2, 64), cache.k.reshape(-1, 2, 64)
        nan = 127 if f8 else np.nan
        v[at[L - n // 2], 0, 5] = nan
        if not f8:
            v[at[L - n // 3 - 1], 0, 9], v[at[L - 1], 1, 7], v[at[L - 1], 1, 8] = np.inf, -np.inf, np.inf
        k[at[L - 1], 0, 3] = nan
    call = Call(ql, ctx, batch, 6, 2, 64, f8, False, cache=cache, spread=0.5)
    call.run()
    call.check()
    call.box.release()


@pytest.mark.parametrize("q16", [False, True])
def test_scores_without_a_number(ql, ctx, q16):
    """Scores of -inf: rows of nothing else are zero, others leave such tokens out. Scores far apart: one token's weight is all."""
    batch = Batch([(1, 40), (70, 70), (1, 700)], 64, seed=2)
    cache = Cache(False, batch.n_page, 64, 1, 64, 2)
    k = cache.k.reshape(-1, 1, 64)
    k[..., 0] = np.abs(k[..., 0]) + 0.5
    for s in range(3):
        at = batch.places(s)
        k[at[::2] if s == 2 else at[:60], 0, 0] = -np.inf
    q = np.abs(np.random.default_rng(1).standard_normal((batch.M, 2, 64))) + 0.5
    call = Call(ql, ctx, batch, 2, 1, 64, False, q16, cache=cache, q=q)
    call.run()
    call.check()
    call.box.release()
    call = Call(ql, ctx, batch, 2, 1, 64, False, q16, spread=300.0)
    call.run()
    call.check()
    call.box.release()


def test_powers_far_apart(ql, ctx):
    """Groups of 16 tokens whose scales lie 2^40 apart, and far from one."""
    batch = Batch([(1, 100), (80, 80), (1, 900)], 64, seed=2)
    cache = Cache(True, batch.n_page, 64, 1, 64, 2)
    g = np.random.default_rng(3)
    cache.scale["v"] *= np.exp2(g.integers(-60, -20, cache.scale["v"].shape)).astype(np.float32)
    cache.scale["k"] *= np.exp2(g.integers(-12, 2, cache.scale["k"].shape)).astype(np.float32)
    call = Call(ql, ctx, batch, 3, 1, 64, True, False, cache=cache)
    call.run()
    call.check()
    call.box.release()


@pytest.mark.parametrize("size", [1e-30, 1e-12, 3e4, 1e30])
def test_sizes_of_q(ql, ctx, size):
    batch = Batch([(1, 100), (80, 80)], 64, seed=2)
    q = np.random.default_rng(4).standard_normal((batch.M, 3, 64)) * size
    k = Cache(False, batch.n_page, 64, 1, 64, 2)
    if size > 1:
        k.k = (k.k / np.float16(256)).astype(np.float16)
    call = Call(ql, ctx, batch, 3, 1, 64, False, False, cache=k, q=q)
    call.run()
    call.check()
    call.box.release()


def test_shared_pages_and_one_page_twice(ql, ctx):
    """Two sequences of one prefix, and a sequence whose list names a page twice."""
    batch = Batch([(1, 200), (30, 150), (1, 190)], 64, seed=2)
    batch.pages[1, :2] = batch.pages[0, :2]
    batch.pages[2, 1] = batch.pages[2, 0]
    call = Call(ql, ctx, batch, 8, 2, 64, True, False)
    call.run()
    call.check()
    call.box.release()


@pytest.mark.parametrize("f8", [False, True])
def test_tables_that_say_what_they_may_not(ql, ctx, f8):
    batch = Batch([(2, 20), (50, 80), (4, 30), (30, 70), (1, 600)], 64, seed=1, pad=2)
    call = Call(ql, ctx, batch, 4, 2, 64, f8, False)
    want = call.want()
    call.desc.max_rows = 40                                                      # the second has more
    lens = batch.kv_len.copy()
    for lens[0], lens[1] in ((1, 80), (batch.max_len + 1, -3), (-2**31, 2**31 - 1)):
        call.box.arena.write(call.box.off("kv_len"), lens)
        call.run()
        call.check(skip=(0, 1), want=want)
    starts = batch.row_start.copy()
    call.box.arena.write(call.box.off("kv_len"), batch.kv_len)
    starts[0] = -4                                                               # the first begins before the batch, the second has too many
    call.box.arena.write(call.box.off("row_start"), starts)
    call.run()
    call.check(skip=(0, 1), want=want)
    call.box.release()
    # pages that are none: their tokens are not seen
    call = Call(ql, ctx, batch, 4, 2, 64, f8, False)
    pages = batch.pages.copy()
    pages[4, [1, 5]] = -1, batch.n_page
    pages[1, 0] = 2**31 - 1
    pages[2, 0] = -9
    call.box.arena.write(call.box.off("pages"), pages)
    call.run()
    got = call.box.get("out")
    assert not got[batch.row_start[2]:batch.row_start[3]].any()                  # nothing is seen: zero
    v, k, q = call.cache.values("v"), call.cache.values("k"), call.q.astype(np.float64)
    for s in (1, 4):
        n, L = batch.seqs[s]
        t = np.arange(L)
        fine = ~np.isin(t // 64, [0] if s == 1 else [1, 5])
        for i in (0, n - 1):
            m, see = batch.row_start[s] + i, fine & (t <= L - n + i)
            at = batch.places(s)[see]
            for h in range(4):
                x = k[at, h // 2] @ q[m, h] / 8
                p = np.exp(x - x.max()) if len(x) else x
                o = p @ v[at, h // 2] / p.sum() if len(x) else np.zeros(64)
                assert np.allclose(got[m, h], o, rtol=0, atol=2.0 ** -15), (s, i, h)
    call.box.release()


def test_bounds_that_are_far(ql, ctx):
    """max_len and max_rows far above what the tables hold give what near ones give, to their tolerance."""
    batch = Batch([(1, 30), (20, 90), (1, 500)], 64, seed=1)
    batch.pages = np.pad(batch.pages, ((0, 0), (0, 600 - batch.max_pages)), constant_values=-1)
    batch.max_pages = 600
    for kw in (dict(max_len=600 * 64, max_rows=5000), dict(max_len=500, max_rows=20), dict(max_len=1100, max_rows=21)):
        call = Call(ql, ctx, batch, 14, 2, 64, False, False, **kw)
        call.run()
        call.check()
        call.box.release()


@pytest.mark.parametrize("D", [64, 128, 48, 112])
@pytest.mark.parametrize("q16", [False, True])
@pytest.mark.parametrize("f8", [False, True])
def test_tiles_in_parts(ql, ctx, f8, q16, D):
    """Bounds so far that tiles have 128 pairs, and so few of them that each is done in parts of its tokens."""
    batch = Batch([(1, 30), (70, 2100), (20, 800), (0, 7)], 256, seed=1, pad=1)
    batch.pages = np.pad(batch.pages, ((0, 0), (0, 2000 - batch.max_pages)), constant_values=-1)
    batch.max_pages = 2000
    call = Call(ql, ctx, batch, 14, 2, D, f8, q16, max_len=2000 * 256)
    call.run()
    call.check()
    call.box.release()


def test_many_sequences(ql, ctx):
    g = np.random.default_rng(2)
    seqs = [(int(n), int(n + p)) for n, p in zip(g.choice([0, 1, 1, 1, 2, 9], 700), g.integers(0, 90, 700))]
    batch = Batch(seqs, 64, seed=1)
    call = Call(ql, ctx, batch, 4, 2, 32, True, False)
    call.run()
    call.check()
    call.box.release()


def test_graph_streams_and_other_calls(ql, ctx):
    """A captured call replayed as lengths change, between other calls of its context; and on another context beside it."""
    batch = Batch([(1, 600), (1, 90), (40, 300), (1, 1400)], 64, seed=4)
    calls = [Call(ql, ctx, batch, 14, 2, 64, f8, False, seed=i) for i, f8 in enumerate((False, True))]
    ctx.graph_begin()
    for c in calls:
        c.run(sync=False) if not c.ql else ctx.paged_attention(c.box.arena, c.box.off("q"), c.dtype, c.box.arena, c.paged, c.desc, batch.M, c.H, c.box.off("out"))
    graph = ctx.graph_end()
    other = ql.Context(0)
    beside = Call(ql, other, Batch([(1, 2000), (30, 700)], 64, seed=8), 28, 4, 128, False, False, seed=8)
    for lens in ([600, 90, 300, 1400], [1, 2, 40, 3], [601, 64, 299, 1399], [600, 90, 300, 1400]):
        for c in calls:
            c.batch.kv_len[:] = lens
            c.batch.seqs = [(n, L) for (n, _), L in zip(batch.seqs, lens)]
            c.box.arena.write(c.box.off("kv_len"), np.array(lens, np.int32))
        graph.launch()
        beside.run(sync=False)
        calls[0].run()
        ctx.sync(), other.sync()
        for c in calls:
            c.check()
        beside.check()
    graph.destroy()
    for c in calls + [beside]:
        c.box.release()
    other.destroy()


@pytest.mark.parametrize("f8", [False, True])
def test_pages_beyond_32_bits(ql, ctx, f8):
    """Keys and values appended to and read from the first and last pages of regions of more than 4 GiB, as from pages of a small cache."""
    KV, D, page, H = 4, 128, 256, 8
    size = KV * page * D * (1 if f8 else 2)
    seqs, far = [(300, 300), (1, 70), (40, 600)], (9 << 29) // size
    batch = Batch(seqs, page, spare=0)
    small = batch.n_page
    g = np.random.default_rng(3)
    box = Box(ql, ctx)
    box.put("q", g.standard_normal((batch.M, H, D)).astype(np.float32))
    for n in "kv":
        box.put(n, g.standard_normal((batch.M, KV, D)).astype(np.float32))
    box.put("qr", np.zeros((batch.M, H, D), np.float32))
    box.put("out", np.zeros((batch.M, H, D), np.float32))
    box.put("table", np.zeros((batch.max_len, D), np.float32))
    batch.put(box)
    box.place()
    ctx.rope_table(box.arena, box.off("table"), batch.max_len, D, 1e4)
    rope = ql.make_rope(box.off("table"), batch.max_len, H, KV, D, cache_dtype=ql.DTYPE_F8 if f8 else ql.DTYPE_F16)
    got = []
    for n_page in (small, far):
        lay = ql.ArenaLayout()
        at = [lay.take(n_page * size), lay.take(n_page * size)] + [lay.take(n_page * KV * page // 16 * 4) for _ in range(2 * f8)]
        cache = ctx.arena(lay.used)
        where = lambda p: np.where(p < small // 2, p, p + n_page - small)  # noqa: E731
        box.arena.write(box.off("pages"), np.where(batch.pages < 0, -1, where(batch.pages)).astype(np.int32))
        for region, bytes_ in zip(at, [size, size, size // D // 4, size // D // 4]):      # zeros, so that what is not appended reads the same
            for p in where(np.arange(small)):
                cache.write(int(region + p * bytes_), np.zeros(bytes_, np.uint8))
        paged = ql.make_paged(at[0], at[1], n_page, page, KV, D, cache_dtype=ql.DTYPE_F8 if f8 else ql.DTYPE_F16,
                              **(dict(k_scale_off=at[2], v_scale_off=at[3]) if f8 else {}))
        desc = batch.desc(ql, box)
        ctx.paged_append(rope, box.arena, box.arena, box.off("q"), box.off("k"), box.off("v"), desc, batch.M, box.off("qr"), ql.DTYPE_F32, cache, paged)
        ctx.paged_attention(box.arena, box.off("qr"), ql.DTYPE_F32, cache, paged, desc, batch.M, H, box.off("out"))
        ctx.sync()
        got.append((box.get("out"), [cache.read(int(at[1] + p * size), (size,), np.uint8) for p in where(np.arange(small))]))
        cache.release()
    (a, pa), (b, pb) = got
    assert a.any() and np.array_equal(a.view(np.uint32), b.view(np.uint32))
    assert all(np.array_equal(x, y) for x, y in zip(pa, pb)) and any(x.any() for x in pa)
    box.release()


def test_refusals(ql, ctx):
    batch = Batch([(3, 60), (1, 9)], 64)
    call = Call(ql, ctx, batch, 4, 2, 64, True, False)
    box = call.box
    size = box.arena.size

    def refused(name, paged={}, desc={}, **kw):
        p, d = (type(s).from_buffer_copy(s) for s in (call.paged, call.desc))
        for s, changes in ((p, paged), (d, desc)):
            for f, v in changes.items():
                setattr(s, f, v)
        a = dict(q=box.off("q"), M=batch.M, H=4, out=box.off("out"), dt=ql.DTYPE_F32)
        a.update(kw)
        with pytest.raises(ql.QlError) as e:
            ctx.paged_attention(box.arena, a["q"], a["dt"], box.arena, p, d, a["M"], a["H"], a["out"])
        assert e.value.name == name, e.value

    for kw in (dict(M=0), dict(M=65536), dict(dt=2), dict(H=0), dict(H=5), dict(H=4098), dict(paged={"cache_dtype": 0}), dict(paged={"page_size": 32}),
               dict(paged={"n_page": -1}), dict(paged={"D": 8}), dict(desc={"n_seq": 0}), dict(desc={"max_len": (1 << 26) + 1, "max_pages": 1 << 30}),
               dict(M=65535, H=256)):
        refused("QL_E_INVALID", **kw)
    for kw in (dict(q=size), dict(out=size - 16), dict(desc={"max_len": 65}), dict(paged={"n_page": 1 << 30}), dict(paged={"v_scale_off": size}),
               dict(desc={"max_pages": 1 << 28, "max_len": 64})):
        refused("QL_E_RANGE", **kw)
    for kw in (dict(q=box.off("q") + 4), dict(out=box.off("out") + 8), dict(paged={"k_off": box.off("K") + 8}), dict(desc={"row_start_off": box.off("row_start") + 1})):
        refused("QL_E_ALIGN", **kw)
    for kw in (dict(out=box.off("q")), dict(out=box.off("K")), dict(out=box.off("V")), dict(out=box.off("pages") & ~15)):
        refused("QL_E_INVALID", **kw)
    assert np.array_equal(box.get("out").view(np.uint32), call.before.view(np.uint32))
    box.release()
    assert f8_encode(np.float64(448)) == 126
