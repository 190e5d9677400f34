"""ql_paged_append against 64-bit arithmetic: positions from the batch's tables, fp16 and e4m3 pages, groups that begin, go on and
grow, what no token is appended to, tables that say what they may not."""
import numpy as np
import pytest

from tests.arena_box import Box
from tests.paged_ref import U, Batch, Cache, f8_decode, power, turned

pytestmark = pytest.mark.gpu
THETA, EPS = 1e4, 1e-6

# sequences (rows, tokens with them)
DECODE = [(1, 1), (1, 16), (1, 17), (1, 64), (1, 65), (1, 200)]
PROMPTS = [(40, 40), (0, 9), (17, 90), (1, 33), (130, 130), (3, 64)]

CASES = [  # seqs, page, H, KV, D, rot, interleaved, norm, f8, q16, strides
    (DECODE, 64, 14, 2, 64, 64, 0, False, False, False, 0),
    (DECODE, 64, 28, 4, 128, 128, 0, True, True, True, 0),
    (PROMPTS, 128, 14, 2, 64, 32, 1, True, True, False, 8),
    (PROMPTS, 64, 6, 3, 128, 64, 0, False, False, True, 0),
    (PROMPTS, 256, 5, 5, 80, 40, 0, True, True, False, 0),
    (PROMPTS, 64, 3, 1, 256, 256, 1, False, True, True, 4),
    (DECODE, 64, 20, 1, 16, 8, 0, True, False, False, 0),
    ([(1, 5)] * 150, 64, 2, 1, 96, 96, 0, False, True, False, 0),
    ([(1000, 1000)], 64, 4, 2, 192, 192, 0, True, True, False, 0),
]


class Call:
    def __init__(self, ql, ctx, batch, H, KV, D, rot, interleaved, norm, f8, q16, gap, seed=1, empty=False, max_pos=None, scale=1.0):
        g = np.random.default_rng(seed)
        self.batch, self.H, self.KV, self.D, self.rot, self.inter, self.q16, self.f8 = batch, H, KV, D, rot, interleaved, q16, f8
        M = batch.M
        self.stride = [h * D + gap for h in (H, KV, KV)]
        self.x = [(scale * g.standard_normal((M, s))).astype(np.float32) for s in self.stride]
        self.norm = [(1 + 0.2 * g.standard_normal(D)).astype(np.float32) for _ in range(2)] if norm else [None, None]
        self.cache = Cache(f8, batch.n_page, batch.page, KV, D, seed, empty)
        self.box = box = Box(ql, ctx)
        for n, x in zip("qkv", self.x):
            box.put(n, x)
        self.before = g.standard_normal((M, H, D)).astype(np.float16 if q16 else np.float32)
        box.put("out", self.before)
        batch.put(box)
        self.cache.put(box)
        self.max_pos = max_pos or batch.max_len
        box.put("table", np.zeros((self.max_pos, rot), np.float32))
        for n, w in zip(("qn", "kn"), self.norm):
            if w is not None:
                box.put(n, w)
        box.place()
        ctx.rope_table(box.arena, box.off("table"), self.max_pos, rot, THETA)
        self.ql, self.ctx = ql, ctx
        self.rope = ql.make_rope(box.off("table"), self.max_pos, H, KV, D, rot_dim=rot, interleaved=bool(interleaved),
                                 q_norm_off=box.off("qn") if norm else None, k_norm_off=box.off("kn") if norm else None, norm_eps=EPS,
                                 q_stride=self.stride[0], k_stride=self.stride[1], v_stride=self.stride[2],
                                 cache_dtype=ql.DTYPE_F8 if f8 else ql.DTYPE_F16)
        self.paged, self.desc = self.cache.desc(ql, box), batch.desc(ql, box)

    def run(self, ctx=None):
        box = self.box
        (ctx or self.ctx).paged_append(self.rope, box.arena, box.arena, box.off("q"), box.off("k"), box.off("v"), self.desc, self.batch.M, box.off("out"),
                                       self.ql.DTYPE_F16 if self.q16 else self.ql.DTYPE_F32, box.arena, self.paged)
        self.ctx.sync()

    def positions(self):
        b, pos = self.batch, np.full(self.batch.M, -1)
        for s, (n, L) in enumerate(b.seqs):
            pos[b.row_start[s]:b.row_start[s] + n] = np.arange(L - n, L)
        return pos

    def heads(self, i):
        return self.x[i][:, :(self.H, self.KV, self.KV)[i] * self.D].reshape(self.batch.M, -1, self.D)

    def check(self, skip=()):
        """what run() has to leave; skip: sequences that have no rows"""
        b, D, pos = self.batch, self.D, self.positions()
        there = pos >= 0
        for s in skip:
            there[b.row_start[s]:b.row_start[s + 1]] = False
        args = (EPS, THETA, self.rot, self.inter)
        want, tol = turned(self.heads(0)[there], pos[there], self.norm[0], *args)
        got = self.box.get("out")
        if self.q16:
            tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        assert np.all(np.abs(got[there] - want) <= tol), np.max(np.abs(got[there] - want) / tol)
        assert np.array_equal(got[~there].view(np.uint8), self.before[~there].view(np.uint8))
        now = self.cache.read(self.box)
        k, k_tol = turned(self.heads(1), np.maximum(pos, 0), self.norm[1], *args)
        v = self.heads(2).astype(np.float64)
        for n, x, e in (("k", k, k_tol), ("v", v, 0 * k_tol)):
            self.check_cache(now, n, x, e, skip)

    def check_cache(self, now, n, x, e, skip):
        b, old, new = self.batch, getattr(self.cache, n), getattr(now, n)
        left = np.ones(old.shape[:2], bool).reshape(-1)                          # tokens that nothing was done to
        grown = np.zeros((left.size // 16, self.KV), bool)
        for s, (rows, L) in enumerate(b.seqs):
            if rows == 0 or s in skip:
                continue
            at, r0 = b.places(s), int(b.row_start[s])
            mine = at[L - rows:]
            left[mine] = False
            flat = new.reshape(-1, self.KV, self.D)
            want, err = x[r0:r0 + rows], e[r0:r0 + rows]
            if not self.f8:
                assert np.all(np.abs(flat[mine].astype(np.float64) - want) <= err + np.abs(want) * 2.0 ** -11 + 2.0 ** -25)
                continue
            scale, was = now.scale[n].reshape(-1, self.KV).astype(np.float64), self.cache.scale[n].reshape(-1, self.KV).astype(np.float64)
            for t0 in range((L - rows) // 16 * 16, L, 16):
                a, z = max(t0, L - rows), min(t0 + 16, L)
                grp = at[a] // 16
                w, we = want[a - (L - rows):z - (L - rows)], err[a - (L - rows):z - (L - rows)]
                top = np.abs(w).max((0, 2))
                slack = we.max((0, 2))
                lo, hi = power(top - slack), power(top + slack)
                if a > t0:
                    lo, hi = np.fmax(lo, was[grp]), np.fmax(hi, was[grp])
                p = scale[grp]
                assert np.all((p == lo) | (p == hi)), (n, s, t0, p, lo, hi)
                got = f8_decode(flat[at[a:z]]) * p[:, None]
                half = np.maximum(np.abs(w) * 2.0 ** -4, 2.0 ** -10 * p[:, None])
                assert np.all(np.abs(got - w) <= half * (1 + 2.0 ** -10) + we)
                if a > t0:                                                       # the group's earlier tokens
                    earlier = at[t0:a]
                    left[earlier] = False
                    was_v = f8_decode(old.reshape(-1, self.KV, self.D)[earlier]) * was[grp][:, None]
                    now_v = f8_decode(flat[earlier]) * p[:, None]
                    small = np.abs(was_v) < 2.0 ** -6 * p[:, None]
                    assert np.all(now_v[~small] == was_v[~small])
                    assert np.all(np.abs(now_v - was_v)[small] <= (2.0 ** -10 * np.broadcast_to(p[:, None], small.shape[1:]))[None].repeat(len(earlier), 0)[small])
                grown[grp] = True
        raw = lambda c: c.view(np.uint8).reshape(left.size, -1)  # noqa: E731
        assert np.array_equal(raw(np.ascontiguousarray(new))[left], raw(np.ascontiguousarray(old))[left])
        if self.f8:
            a, z = now.scale[n].reshape(-1, self.KV), self.cache.scale[n].reshape(-1, self.KV)
            assert np.array_equal(a[~grown].view(np.uint32), z[~grown].view(np.uint32))


@pytest.mark.parametrize("case", range(len(CASES)))
def test_append(ql, ctx, case):
    seqs, page, *rest = CASES[case]
    call = Call(ql, ctx, Batch(seqs, page, seed=case, pad=3), *rest)
    call.run()
    call.check()
    call.box.release()


@pytest.mark.parametrize("f8", [False, True])
def test_append_to_memory_that_holds_anything(ql, ctx, f8):
    """A prompt into pages of NaN, then its next tokens one by one: each group's scale comes from its own tokens."""
    batch = Batch([(37, 37), (16, 16)], 64, seed=4)
    call = Call(ql, ctx, batch, 4, 2, 64, 64, 0, False, f8, False, 0, empty=True, max_pos=64)
    call.run()
    now = call.cache.read(call.box)
    for s, (n, L) in enumerate(batch.seqs):
        for x in ("k", "v"):
            assert np.isfinite(now.values(x)[batch.places(s)]).all()
    rest = np.setdiff1d(np.arange(batch.n_page * 64), np.concatenate([batch.places(s) for s in range(2)]))
    assert np.isnan((f8_decode(now.k) if f8 else now.k).reshape(-1, 2, 64)[rest].astype(np.float64)).all()
    call.box.release()


def test_group_grows(ql, ctx):
    """Tokens of growing size, one a pass: earlier ones keep their values where e4m3 can hold them under the new scale."""
    steps, D = 40, 64
    g = np.random.default_rng(8)
    v = (g.standard_normal((steps, D)) * 1.7 ** np.arange(steps)[:, None] * 1e-3).astype(np.float32)
    box = Box(ql, ctx)
    cache = Cache(True, Batch([(1, 1)], 64).n_page, 64, 1, D, empty=True)
    cache.put(box)
    for n in "qk":
        box.put(n, np.zeros((1, D), np.float32))
    for t in range(steps):
        box.put(f"v{t}", v[t:t + 1])
        Batch([(1, t + 1)], 64).put(box, str(t))
    box.put("out", np.zeros((1, D), np.float32))
    box.put("table", np.zeros((64, D), np.float32))
    box.place()
    ctx.rope_table(box.arena, box.off("table"), 64, D, THETA)
    rope = ql.make_rope(box.off("table"), 64, 1, 1, D, cache_dtype=ql.DTYPE_F8)
    b = Batch([(1, 1)], 64)
    moved = np.zeros((steps, D))
    scale = np.zeros(3)
    for t in range(steps):
        ctx.paged_append(rope, box.arena, box.arena, box.off("q"), box.off("k"), box.off(f"v{t}"),
                         b.desc(ql, box, str(t), max_len=t + 1), 1, box.off("out"), ql.DTYPE_F32, box.arena, cache.desc(ql, box))
        ctx.sync()
        now = cache.read(box)
        grp, at = t // 16, int(b.pages[0, 0]) * 64
        p = power(np.abs(v[t]).max())
        p = p if t % 16 == 0 else max(p, scale[grp])
        assert now.scale["v"].reshape(-1)[at // 16 + grp] == p
        scale[grp] = p
        from tests.paged_ref import f8_encode
        moved[16 * grp:t] = f8_decode(f8_encode(moved[16 * grp:t] / p)) * p
        moved[t] = f8_decode(f8_encode(v[t] / p)) * p
        assert np.array_equal(now.values("v")[at:at + t + 1, 0], moved[:t + 1])
    box.release()


def test_values_that_are_not_finite(ql, ctx):
    batch = Batch([(20, 20)], 64)
    call = Call(ql, ctx, batch, 2, 1, 64, 64, 0, False, True, False, 0)
    x = call.x[2]
    x[3, 5], x[4, 6], x[18, 7] = np.inf, -np.inf, np.nan
    call.box.arena.write(call.box.off("v"), x)
    call.run()
    now = call.cache.read(call.box).values("v")[batch.places(0), 0]
    bad = ~np.isfinite(x)
    assert np.isnan(now[bad]).all() and np.isfinite(now[~bad]).all()
    p = power(np.abs(np.where(bad, 0, x))[:16].max())
    assert call.cache.read(call.box).scale["v"].reshape(-1)[batch.places(0)[0] // 16] == p
    call.box.release()


@pytest.mark.parametrize("f8", [False, True])
def test_tables_that_say_what_they_may_not(ql, ctx, f8):
    """Sequences too long, with too many rows, of descending rows or with pages that are none: skipped, nothing else changes."""
    batch = Batch([(2, 20), (5, 40), (4, 30), (3, 70)], 64, pad=2)
    call = Call(ql, ctx, batch, 4, 2, 64, 64, 0, True, f8, False, 0)
    call.desc.max_rows = 4                                                       # the second has more
    lens = batch.kv_len.copy()
    lens[0] = 1                                                                  # fewer tokens than rows
    call.box.arena.write(call.box.off("kv_len"), lens)
    pages = batch.pages.copy()
    call.box.arena.write(call.box.off("pages"), pages)
    call.run()
    call.check(skip=(0, 1))
    lens[0] = batch.max_len + 1                                                  # longer than max_len
    lens[1] = -5
    call.box.arena.write(call.box.off("kv_len"), lens)
    call.run()
    call.check(skip=(0, 1))
    call.box.release()
    # no page there: the rows of q are turned, the tokens not stored
    call = Call(ql, ctx, batch, 4, 2, 64, 64, 0, True, f8, False, 0)
    pages[:] = [[batch.n_page, 0], [-1, 0], [2**31 - 1, 0], [-2**31, -2**31]]
    call.box.arena.write(call.box.off("pages"), pages)
    call.run()
    now = call.cache.read(call.box)
    assert np.array_equal(now.k.view(np.uint8), call.cache.k.view(np.uint8)) and np.array_equal(now.v.view(np.uint8), call.cache.v.view(np.uint8))
    call.box.release()


def test_in_place_and_other_streams(ql, ctx):
    """q turned where it lies; two contexts on their own batches at once; a captured graph replayed as the tables change."""
    batch = Batch([(3, 60), (1, 9)], 64)
    call = Call(ql, ctx, batch, 4, 2, 64, 64, 0, False, True, False, 0)
    box = call.box
    for i in range(2):
        ctx.paged_append(call.rope, box.arena, box.arena, box.off("q"), box.off("k"), box.off("v"), call.desc, batch.M, box.off("q"), ql.DTYPE_F32,
                         box.arena, call.paged)
        ctx.sync()
        want, tol = turned(call.heads(0), call.positions(), None, EPS, THETA, 64, 0)
        assert np.all(np.abs(box.get("q").reshape(want.shape) - want) <= tol)
        box.arena.write(box.off("q"), call.x[0])
    ctx.graph_begin()
    ctx.paged_append(call.rope, box.arena, box.arena, box.off("q"), box.off("k"), box.off("v"), call.desc, batch.M, box.off("out"), ql.DTYPE_F32,
                     box.arena, call.paged)
    graph = ctx.graph_end()
    call.desc.max_len = 64
    for lens in ([60, 9], [50, 20], [33, 17]):
        batch.kv_len[:] = lens
        batch.seqs = [(3, lens[0]), (1, lens[1])]
        box.arena.write(box.off("kv_len"), batch.kv_len)
        call.cache = call.cache.read(box)
        graph.launch()
        ctx.sync()
        call.check()
    graph.destroy()
    box.release()
    other = ql.Context(0)
    calls = [Call(ql, c, Batch(DECODE, 64, seed=i), 14, 2, 64, 64, 0, False, bool(i), False, 0, seed=i) for i, c in enumerate((ctx, other))]
    for c in calls:
        b = c.box
        c.ctx.paged_append(c.rope, b.arena, b.arena, b.off("q"), b.off("k"), b.off("v"), c.desc, c.batch.M, b.off("out"), ql.DTYPE_F32, b.arena, c.paged)
    for c in calls:
        c.ctx.sync()
    for c in calls:
        c.check()
        c.box.release()
    other.destroy()


def test_refusals(ql, ctx):
    batch = Batch([(3, 60), (1, 9)], 64)
    call = Call(ql, ctx, batch, 4, 2, 64, 64, 0, False, True, False, 0)
    box = call.box
    size = box.arena.size

    def refused(name, rope={}, paged={}, desc={}, **kw):
        r, p, d = (type(s).from_buffer_copy(s) for s in (call.rope, call.paged, call.desc))
        for s, changes in ((r, rope), (p, paged), (d, desc)):
            for f, v in changes.items():
                setattr(s, f, v)
        a = dict(q=box.off("q"), k=box.off("k"), v=box.off("v"), M=batch.M, out=box.off("out"), dt=ql.DTYPE_F32)
        a.update(kw)
        with pytest.raises(ql.QlError) as e:
            ctx.paged_append(r, box.arena, box.arena, a["q"], a["k"], a["v"], d, a["M"], a["out"], a["dt"], box.arena, p)
        assert e.value.name == name, e.value

    for kw in (dict(M=0), dict(M=65536), dict(dt=2), dict(rope={"n_head": 0}), dict(rope={"rot_dim": 12}), dict(rope={"rot_dim": 72}), dict(rope={"interleaved": 2}),
               dict(rope={"q_stride": 6}), dict(rope={"norm_eps": float("nan")}), dict(rope={"n_kv_head": 1}), dict(rope={"cache_dtype": ql.DTYPE_F16}),
               dict(paged={"cache_dtype": 0}), dict(paged={"page_size": 32}), dict(paged={"page_size": 96}), dict(paged={"n_page": 0}), dict(paged={"D": 72}),
               dict(paged={"D": 272}), dict(paged={"reserved": 1}), dict(paged={"n_kv_head": 0}), dict(desc={"n_seq": 0}), dict(desc={"n_seq": 4097}),
               dict(desc={"max_rows": 0}), dict(desc={"max_len": 0}), dict(desc={"max_pages": 0})):
        refused("QL_E_INVALID", **kw)
    for kw in (dict(q=size), dict(out=size - 16), dict(desc={"max_len": 64 * batch.max_pages + 1}), dict(desc={"max_len": 61}), dict(paged={"n_page": 1 << 30}),
               dict(paged={"k_scale_off": size}), dict(desc={"pages_off": size}), dict(desc={"row_start_off": size - 4}), dict(rope={"table_off": size - 64})):
        refused("QL_E_RANGE", **kw)
    for kw in (dict(q=box.off("q") + 4), dict(out=box.off("out") + 8), dict(paged={"v_off": box.off("V") + 8}), dict(paged={"v_scale_off": box.off("vs") + 4}),
               dict(desc={"kv_len_off": box.off("kv_len") + 2}), dict(rope={"table_off": box.off("table") + 4})):
        refused("QL_E_ALIGN", **kw)
    for kw in (dict(out=box.off("k")), dict(out=box.off("q") + 16), dict(paged={"v_off": box.off("K") + 16}), dict(paged={"k_scale_off": box.off("vs")}),
               dict(paged={"k_off": box.off("V") - 16}), dict(out=box.off("q"), dt=ql.DTYPE_F16),
               dict(v=box.off("V"))):
        refused("QL_E_INVALID", **kw)
    now = call.cache.read(box)
    assert np.array_equal(now.k, call.cache.k) and np.array_equal(box.get("out").view(np.uint32), call.before.view(np.uint32))
    box.release()
    assert U == np.finfo(np.float32).eps / 2
