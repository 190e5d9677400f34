"""ql_lora_add against 64-bit arithmetic: adapters of many rows in any order, rows without one, several projections, ranks and sizes,
in place and apart."""
import numpy as np
import pytest

from tests.arena_box import Box
from tests.paged_ref import U

pytestmark = pytest.mark.gpu


class Call:
    """targets: (K, N, rank, n) each; same: all read the first one's x"""

    def __init__(self, ql, ctx, M, targets, x16, ids, seed=1, same=False, place=False, scales=True):
        g = np.random.default_rng(seed)
        self.ql, self.ctx, self.M, self.targets, self.x16, self.place, self.scales = ql, ctx, M, targets, x16, place, scales
        self.ids = np.asarray(ids, np.int32)
        self.box = box = Box(ql, ctx)
        box.put("ids", self.ids)
        self.x, self.a, self.b, self.base, self.scale = [], [], [], [], []
        for i, (K, N, r, n) in enumerate(targets):
            self.x.append(self.x[0] if same and i else g.standard_normal((M, K)).astype(np.float16 if x16 else np.float32))
            self.a.append((g.standard_normal((n, r, K)) * K ** -0.5).astype(np.float16))
            self.b.append((g.standard_normal((n, N, r)) * r ** -0.5).astype(np.float16))
            self.base.append(g.standard_normal((M, N)).astype(np.float32))
            self.scale.append(g.uniform(0.5, 2, n).astype(np.float32))
            if not (same and i):
                box.put(f"x{i}", self.x[i])
            box.put(f"a{i}", self.a[i]), box.put(f"b{i}", self.b[i]), box.put(f"s{i}", self.scale[i])
            box.put(f"base{i}", self.base[i])
            if not place:
                box.put(f"y{i}", np.full((M, N), np.nan, np.float32))
        box.place()
        self.xo = [box.off("x0" if same else f"x{i}") for i in range(len(targets))]
        self.descs = [ql.make_lora(box.off(f"a{i}"), box.off(f"b{i}"), K, N, r, n, scale_off=box.off(f"s{i}") if scales else None)
                      for i, (K, N, r, n) in enumerate(targets)]

    def out(self, i):
        return f"base{i}" if self.place else f"y{i}"

    def run(self, ctx=None, sync=True):
        box, n = self.box, range(len(self.targets))
        c = ctx or self.ctx
        c.lora_add(self.descs, box.arena, box.arena, box.off("ids"), self.xo, self.ql.DTYPE_F16 if self.x16 else self.ql.DTYPE_F32, self.M,
                   [box.off(f"base{i}") for i in n], [box.off(self.out(i)) for i in n])
        if sync:
            c.sync()

    def check(self):
        got_all = []
        for i, (K, N, r, n) in enumerate(self.targets):
            got = self.box.get(self.out(i))
            got_all.append(got)
            want, tol = self.base[i].astype(np.float64), np.zeros((self.M, N))
            has = (self.ids >= 0) & (self.ids < n)
            for k in np.unique(self.ids[has]):
                m = self.ids == k
                x, a, b = (v.astype(np.float64) for v in (self.x[i][m], self.a[i][k], self.b[i][k]))
                s = float(self.scale[i][k]) if self.scales else 1.0
                want[m] += s * (x @ a.T) @ b.T
                # fp32 sums of K and of r products, each off by as many u of the products' sizes at most, and the scale's product; many rows:
                # x's and t's two parts carry 2^-22 of the largest of their 64 columns, or of the row's ranks
                tol[m] = s * ((K + 4) * U * (np.abs(x) @ np.abs(a).T) + (r + 4) * U * np.abs(x @ a.T)) @ np.abs(b).T
            tol += 2 * U * np.abs(want)
            with np.errstate(invalid="ignore"):
                assert np.all(np.abs(got - want)[has] <= tol[has]), (i, np.nanmax(np.abs(got - want)[has] / tol[has]))
            assert np.array_equal(got[~has].view(np.uint32), self.base[i][~has].view(np.uint32))
        return got_all


CASES = [  # M, targets, how the ids lie
    (1, [(896, 896, 8, 1)], "mixed"),
    (1, [(896, 128, 16, 3), (896, 128, 16, 3)], "none"),
    (4, [(896, 896, 8, 3), (896, 128, 8, 3), (896, 128, 8, 3)], "mixed"),
    (16, [(1000, 100, 24, 16)], "each"),
    (17, [(64, 4, 64, 40)], "mixed"),
    (33, [(8, 1000, 128, 2)], "mixed"),
    (64, [(3584, 3584, 16, 24), (3584, 512, 16, 24)], "mixed"),
    (70, [(4864, 896, 32, 5)], "runs"),
    (200, [(896, 4864, 64, 4), (896, 4864, 64, 4)], "runs"),
    (300, [(520, 260, 40, 7)], "mixed"),
    (1000, [(896, 128, 16, 6)], "runs"),
    (130, [(2056, 12, 96, 3)], "one"),
    (1500, [(904, 300, 64, 9), (904, 20, 24, 9)], "mixed"),
    (1030, [(72, 516, 8, 2)], "runs"),
    (1100, [(200, 60, 72, 3), (200, 20, 24, 3)], "mixed"),                       # tiles of 32 rows, groups of ranks that end inside
    (2000, [(64, 36, 128, 5)] * 4, "runs"),                                      # more tiles of ranks than a launch has
    (1024, [(264, 256, 48, 3), (264, 260, 16, 3)], "runs"),
    (20000, [(16, 8, 128, 3)] * 8, "runs"),                                      # more rows than the workspace has room for at once
]


def ids_of(how, M, n, seed=3):
    g = np.random.default_rng(seed)
    if how == "none":
        return np.full(M, -1)
    if how == "one":
        return np.full(M, n - 1)
    if how == "each":
        return g.permutation(M) % n
    ids = g.integers(-1, n, M)
    return np.sort(ids) if how == "runs" else ids


@pytest.mark.parametrize("x16", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_lora(ql, ctx, case, x16):
    M, targets, how = CASES[case]
    same = len({t[0] for t in targets}) == 1
    call = Call(ql, ctx, M, targets, x16, ids_of(how, M, targets[0][3]), same=same, scales=case % 2 == 0)
    call.run()
    first = call.check()
    call.run()
    assert all(np.array_equal(call.box.get(call.out(i)).view(np.uint32), y.view(np.uint32)) for i, y in enumerate(first))
    call.box.release()
    call = Call(ql, ctx, M, targets, x16, ids_of(how, M, targets[0][3], 5), place=True)
    call.run()
    call.check()
    call.box.release()


def test_ids_that_are_none(ql, ctx):
    """Ids outside an adapter's number are rows without one, also where projections have different numbers."""
    ids = [0, 5, -1, 2**31 - 1, -2**31, 4, 3, 1]
    call = Call(ql, ctx, 8, [(64, 64, 8, 5), (64, 32, 16, 2)], False, ids)
    call.run()
    call.check()
    call.box.release()


@pytest.mark.parametrize("M", [40, 600])
def test_rows_apart(ql, ctx, M):
    """A row that is not finite, its adapter's too, stays with itself: every other row has the bits that it has without."""
    ids = np.arange(M) % 3
    call = Call(ql, ctx, M, [(256, 64, 16, 3)], False, ids)
    call.run()
    plain = call.check()[0]
    x = call.x[0].copy()
    x[7, 3], x[20, 9], x[21, 1] = np.nan, np.inf, 3e38
    call.box.arena.write(call.xo[0], x)
    a = call.a[0].copy()
    a[2, 3, 5] = np.nan
    call.box.arena.write(call.box.off("a0"), a)
    call.run()
    got = call.box.get("y0")
    rest = ~np.isin(np.arange(M), (7, 20, 21)) & (ids != 2)
    assert np.array_equal(got[rest].view(np.uint32), plain[rest].view(np.uint32))
    assert np.isnan(got[7]).all() and not np.isfinite(got[20]).any() and np.isnan(got[ids == 2]).all()
    call.box.release()


def test_rows_apart_in_tiles_of_32(ql, ctx):
    ids = np.arange(1300) % 3
    call = Call(ql, ctx, 1300, [(256, 64, 48, 3)], True, ids)
    call.run()
    plain = call.check()[0]
    x = call.x[0].copy()
    x[7, 3], x[1220, 9], x[1299, 255] = np.nan, np.inf, np.nan
    call.box.arena.write(call.xo[0], x)
    b = call.b[0].copy()
    b[1, 3, 5] = np.nan
    call.box.arena.write(call.box.off("b0"), b)
    call.run()
    got = call.box.get("y0")
    rest = ~np.isin(np.arange(1300), (7, 1220, 1299))
    other = np.arange(64) != 3
    assert np.array_equal(got[rest][:, other].view(np.uint32), plain[rest][:, other].view(np.uint32))
    assert np.isnan(got[7]).all() and np.isnan(got[1299]).all() and not np.isfinite(got[1220]).any()
    assert np.array_equal(np.isnan(got[rest][:, 3]), ids[rest] == 1)
    call.box.release()


@pytest.mark.parametrize("M", [3, 100, 600])
def test_sizes_of_x(ql, ctx, M):
    """fp32 rows of any size keep fp32's accuracy."""
    call = Call(ql, ctx, M, [(256, 64, 16, 3)], False, np.arange(M) % 3)
    for size in (1e-30, 1e-8, 1e6, 1e25):
        x = (np.random.default_rng(1).standard_normal((M, 256)) * size * np.exp2(np.random.default_rng(2).integers(-20, 1, (M, 256)))).astype(np.float32)
        call.x[0] = x
        call.box.arena.write(call.xo[0], x)
        call.base[0][:] = 0
        call.box.arena.write(call.box.off("base0"), call.base[0])
        call.run()
        call.check()
    call.box.release()


def test_graph_streams_and_other_calls(ql, ctx):
    calls = [Call(ql, ctx, M, [(896, 896, 16, 6), (896, 128, 16, 6)], False, ids_of("mixed", M, 6), same=True, seed=M) for M in (5, 90, 700)]
    ctx.graph_begin()
    for c in calls:
        c.run(sync=False)
    graph = ctx.graph_end()
    other = ql.Context(0)
    beside = Call(ql, other, 300, [(896, 896, 32, 4)], False, ids_of("runs", 300, 4))
    for step in range(3):
        for c in calls:
            c.ids = ids_of("mixed", c.M, 6, seed=step).astype(np.int32)
            c.box.arena.write(c.box.off("ids"), c.ids)
        graph.launch()
        beside.run(sync=False)
        calls[1].run(sync=False)
        ctx.sync(), other.sync()
        for c in calls + [beside]:
            c.check()
    graph.destroy()
    for c in calls + [beside]:
        c.box.release()
    other.destroy()


def test_refusals(ql, ctx):
    call = Call(ql, ctx, 6, [(64, 32, 8, 3), (64, 16, 8, 3)], False, [0, 1, 2, -1, 0, 1], same=True)
    box = call.box
    size = box.arena.size
    before = [box.get(call.out(i)) for i in range(2)]

    def refused(name, desc={}, **kw):
        d = [type(s).from_buffer_copy(s) for s in call.descs]
        for f, v in desc.items():
            setattr(d[1], f, v)
        a = dict(descs=d, ids=box.off("ids"), x=call.xo, dt=ql.DTYPE_F32, M=6, base=[box.off("base0"), box.off("base1")], y=[box.off("y0"), box.off("y1")])
        a.update(kw)
        with pytest.raises(ql.QlError) as e:
            ctx.lora_add(a["descs"], box.arena, box.arena, a["ids"], a["x"], a["dt"], a["M"], a["base"], a["y"])
        assert e.value.name == name, e.value

    y0, y1 = box.off("y0"), box.off("y1")
    for kw in (dict(desc={"K": 60}), dict(desc={"K": 0}), dict(desc={"N": 6}), dict(desc={"N": -4})):
        refused("QL_E_DIMS", **kw)
    for kw in (dict(M=0), dict(M=65536), dict(dt=2), dict(dt=-1), dict(desc={"rank": 12}), dict(desc={"rank": 0}), dict(desc={"rank": 136}), dict(desc={"n_adapter": 0}),
               dict(descs=[], x=[], base=[], y=[]), dict(descs=[call.descs[0]] * 9, x=[call.xo[0]] * 9, base=[y0] * 9, y=[y0] * 9),
               dict(y=[y0, y0]), dict(y=[y0, y0 + 16]), dict(y=[y0, box.off("base0")]), dict(y=[y0, box.off("base1") + 16]), dict(y=[call.xo[0], y1]),
               dict(y=[y0, box.off("a1")]), dict(y=[box.off("ids") // 16 * 16, y1])):
        refused("QL_E_INVALID", **kw)
    for kw in (dict(ids=size), dict(x=[call.xo[0], size - 32]), dict(base=[size, size]), dict(y=[y0, size - 64]), dict(desc={"a_off": size}), dict(desc={"n_adapter": 65536}),
               dict(desc={"scale_off": size})):
        refused("QL_E_RANGE", **kw)
    for kw in (dict(ids=box.off("ids") + 2), dict(x=[call.xo[0], call.xo[0] + 4]), dict(y=[y0, y1 + 4]), dict(base=[y0, box.off("base1") + 8]),
               dict(desc={"a_off": box.off("a1") + 2}), dict(desc={"scale_off": box.off("s1") + 2})):
        refused("QL_E_ALIGN", **kw)
    with pytest.raises(ValueError):
        ctx.lora_add(call.descs, box.arena, box.arena, box.off("ids"), call.xo, 0, 6, [0], [0, 0])
    assert all(np.array_equal(box.get(call.out(i)).view(np.uint32), b.view(np.uint32)) for i, b in enumerate(before))
    box.release()
