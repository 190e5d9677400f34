"""GPU: norms of the query and key heads, rotation and cache store (ql_qk_norm_rope, ql_rope_table) against the formula in 64
bits. Rounding, in units u = 2^-24 of an fp32 step's half: the head's mean square has up to 8 + 32 added terms, half of
whose error reaches the norm (20 u), the root, the division and the two products 5 u, the angle's cosine and sine 1 u, the
rotation's products and sum 3 u: at most 32 u of |a cos| + |b sin|, and for an fp16 cache half a step of fp16 (2^-11; 2^-25 below
its normal range)."""
import numpy as np
import pytest

from tests.arena_box import Box

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def angles(pos, rot, theta):
    t = np.asarray(pos, np.float64)[:, None] * theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    return np.cos(t), np.sin(t)


def pairs(rot, interleaved):
    return (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2, rot))


def formula(x, w, eps, c, s, rot, interleaved):
    """(values, what their rounding is measured by) of [M, heads, D]."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, size = x.copy(), np.abs(x)
    i, j = pairs(rot, interleaved)
    c, s = c[:, None, :], s[:, None, :]
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size[..., i] = np.abs(x[..., i] * c) + np.abs(x[..., j] * s)
    size[..., j] = np.abs(x[..., j] * c) + np.abs(x[..., i] * s)
    return y, size


CASES = [
    # M, H, KV, D, rot, interleaved, norms, fp16 cache, fused rows, slot0, label
    (1, 14, 2, 64, 64, False, "", False, False, 0, "one token of the small model"),
    (3, 28, 4, 128, 128, False, "qk", True, False, 5, "normed heads, half cache"),
    (17, 28, 4, 128, 128, True, "qk", False, True, 2, "interleaved pairs, rows of one projection"),
    (5, 6, 3, 80, 80, False, "qk", True, True, 1, "a head of 10 lanes"),
    (4, 3, 1, 96, 32, False, "k", False, False, 0, "partial rotation, only keys normed"),
    (2, 5, 5, 8, 8, True, "q", True, False, 3, "the smallest head, only queries normed"),
    (9, 2, 1, 256, 128, True, "qk", False, True, 7, "the largest head, partial and interleaved"),
    (33, 1, 1, 24, 8, False, "qk", True, False, 0, "three lanes a head, one head"),
    (300, 4, 2, 16, 16, False, "", False, False, 11, "many rows, two lanes a head"),
]


def setup(ql, ctx, M, H, KV, D, rot, interleaved, norms, half, fused, slot0, seed=1, pos=None, theta=1e4, max_pos=700, extra=5):
    g = np.random.default_rng(seed)
    d = {"q": g.standard_normal((M, H * D)), "k": g.standard_normal((M, KV * D)), "v": g.standard_normal((M, KV * D))}
    d = {n: a.astype(np.float32) for n, a in d.items()}
    pos = g.integers(0, max_pos, M).astype(np.int32) if pos is None else np.asarray(pos, np.int32)
    T = slot0 + M + extra
    t = np.float16 if half else np.float32
    w, act, cache = Box(ql, ctx), Box(ql, ctx), Box(ql, ctx)
    w.put("table", np.zeros((max_pos, rot), np.float32))
    d["qn"], d["kn"] = (1 + 0.3 * g.standard_normal((2, D))).astype(np.float32)
    w.put("qn", d["qn"])
    w.put("kn", d["kn"])
    if fused:
        base = act.put("qkv", np.concatenate([d["q"], d["k"], d["v"]], 1))
        offs = [base, base + 4 * H * D, base + 4 * (H + KV) * D]
        stride = (H + 2 * KV) * D
    else:
        offs, stride = [act.put(n, d[n]) for n in "qkv"], 0
    act.put("pos", pos)
    act.put("out", np.full((M + 1, H * D), 7, np.float32))
    for n in "kv":
        cache.put(n, np.full((T, KV * D), 9, t))
    for b in (w, act, cache):
        b.place()
    ctx.rope_table(w.arena, w.off("table"), max_pos, rot, theta)
    desc = ql.make_rope(w.off("table"), max_pos, H, KV, D, rot_dim=rot, interleaved=interleaved, q_norm_off=w.off("qn") if "q" in norms else None,
                        k_norm_off=w.off("kn") if "k" in norms else None, norm_eps=1e-5, q_stride=stride, k_stride=stride, v_stride=stride,
                        cache_dtype=ql.DTYPE_F16 if half else ql.DTYPE_F32)
    args = [desc, w.arena, act.arena, *offs, act.off("pos"), M, act.off("out"), cache.arena, cache.off("k"), cache.off("v"), T, slot0]
    return d, pos, (w, act, cache), args


def check(d, pos, boxes, M, H, KV, D, rot, interleaved, norms, half, slot0, theta=1e4, rows=None, q_name="out"):
    _, act, cache = boxes
    rows = np.arange(M) if rows is None else rows
    c, s = angles(pos, rot, theta)
    got = {"q": act.get(q_name)[:M].reshape(M, H, D), "k": cache.get("k")[slot0:slot0 + M].reshape(M, KV, D),
           "v": cache.get("v")[slot0:slot0 + M].reshape(M, KV, D)}
    for n, heads in (("q", H), ("k", KV), ("v", KV)):
        x = d[n].reshape(M, heads, D)
        if n == "v":
            want, size = x.astype(np.float64), np.zeros(x.shape)
        else:
            want, size = formula(x, d["qn" if n == "q" else "kn"].astype(np.float64) if n in norms else None, 1e-5, c, s, rot, interleaved)
        tol = 32 * U * size
        if half and n != "q":
            tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
        off = np.abs(got[n].astype(np.float64) - want)[rows] - tol[rows]
        assert off.max() <= 0, (n, off.max())


@pytest.mark.parametrize("M,H,KV,D,rot,interleaved,norms,half,fused,slot0,label", CASES)
def test_rope_matches_formula(ql, ctx, M, H, KV, D, rot, interleaved, norms, half, fused, slot0, label):
    print(label, flush=True)
    d, pos, boxes, args = setup(ql, ctx, M, H, KV, D, rot, interleaved, norms, half, fused, slot0)
    ctx.qk_norm_rope(*args)
    check(d, pos, boxes, M, H, KV, D, rot, interleaved, norms, half, slot0)
    w, act, cache = boxes
    assert (act.get("out")[M:] == 7).all()                                   # what lies behind stays
    for n in "kv":
        kept = cache.get(n)
        assert (kept[:slot0] == 9).all() and (kept[slot0 + M:] == 9).all()
    for b in boxes:
        b.release()


def test_table_is_rounded_once(ql, ctx):
    """Far positions: the angle is formed in 64 bits, so every cosine and sine is within half a step (one more where fp64's own
    library rounds the other way: 2^-29 of it)."""
    max_pos, rot, theta = 200000, 16, 1e6
    w = Box(ql, ctx)
    w.put("table", np.zeros((max_pos, rot), np.float32))
    w.place()
    ctx.rope_table(w.arena, w.off("table"), max_pos, rot, theta)
    c, s = angles(np.arange(max_pos), rot, theta)
    want = np.concatenate([c, s], 1)
    # angles up to 2e5 in fp64: 2e5 * 2^-53 * 3 absolute
    assert (np.abs(w.get("table") - want) <= np.abs(want) * U * (1 + 2.0 ** -20) + 2e5 * 2.0 ** -51).all()
    w.release()


@pytest.mark.parametrize("half", [False, True])
def test_padding_rows_are_left_out(ql, ctx, half):
    M, H, KV, D, rot = 6, 4, 2, 32, 32
    pos = [3, -1, 699, 700, 2**31 - 1, 0]
    d, pos, boxes, args = setup(ql, ctx, M, H, KV, D, rot, False, "qk", half, False, 2, pos=pos)
    ctx.qk_norm_rope(*args)
    there = np.array([0, 2, 5])
    safe = np.where((pos >= 0) & (pos < 700), pos, 0)
    check(d, safe, boxes, M, H, KV, D, rot, False, "qk", half, 2, rows=there)
    for m in (1, 3, 4):
        assert (boxes[1].get("out")[m] == 7).all() and (boxes[2].get("k")[2 + m] == 9).all() and (boxes[2].get("v")[2 + m] == 9).all()
    for b in boxes:
        b.release()


def test_in_place(ql, ctx):
    M, H, KV, D, rot = 7, 5, 1, 64, 48
    d, pos, boxes, args = setup(ql, ctx, M, H, KV, D, rot, False, "qk", False, False, 0)
    args[8] = args[3]
    ctx.qk_norm_rope(*args)
    check(d, pos, boxes, M, H, KV, D, rot, False, "qk", False, 0, q_name="q")
    for b in boxes:
        b.release()


def test_offsets_past_32_bits(ql, ctx):
    """The last slots of a half cache of 4.5 GiB a region."""
    M, H, KV, D = 3, 2, 8, 256
    T = (9 << 29) // (KV * D * 2) + 5
    d, pos, boxes, args = setup(ql, ctx, M, H, KV, D, D, False, "", True, False, 0)
    big = ctx.arena(T * KV * D * 2)
    small = Box(ql, ctx)
    args[9:] = [big, 0, 0, T, T - M]
    with pytest.raises(ql.QlError):                                          # K and V in one region
        ctx.qk_norm_rope(*args)
    other = ctx.arena(T * KV * D * 2 * 2)
    big.release()
    args[9:] = [other, 0, T * KV * D * 2, T, T - M]
    ctx.qk_norm_rope(*args)
    c, s = angles(pos, D, 1e4)
    want, size = formula(d["k"].reshape(M, KV, D), None, 0, c, s, D, False)
    got = other.read((T - M) * KV * D * 2, (M, KV, D), np.float16).astype(np.float64)
    assert (np.abs(got - want) <= 32 * U * size + 2.0 ** -11 * np.abs(want) + 2.0 ** -25).all()
    got = other.read((2 * T - M) * KV * D * 2, (M, KV, D), np.float16)
    assert np.array_equal(got, d["v"].reshape(M, KV, D).astype(np.float16))
    other.release()
    for b in boxes:
        b.release()
    del small


def test_refusals(ql, ctx):
    M, H, KV, D, rot = 4, 4, 2, 32, 32
    d, pos, boxes, args = setup(ql, ctx, M, H, KV, D, rot, False, "qk", False, False, 2)
    w, act, cache = boxes

    def refused(name, **change):
        a = list(args)
        desc = ql.RopeDesc.from_buffer_copy(a[0])
        for key, v in change.items():
            if isinstance(key, str) and hasattr(desc, key):
                setattr(desc, key, v)
        a[0] = desc
        for i, v in change.get("at", {}).items():
            a[i] = v
        with pytest.raises(ql.QlError) as e:
            ctx.qk_norm_rope(*a)
        assert e.value.name == name, (change, e.value)

    for change in ({"D": 12}, {"D": 264}, {"D": 0}, {"rot_dim": 0}, {"rot_dim": 12}, {"rot_dim": 40}, {"n_head": 0}, {"n_kv_head": 0}, {"max_pos": 0},
                   {"interleaved": 2}, {"cache_dtype": 2}, {"norm_eps": -1.0}, {"norm_eps": float("nan")}, {"q_stride": 64}, {"k_stride": -64},
                   {"v_stride": 66}, {"reserved": 1}, {"at": {7: 0}}, {"at": {7: 65536}}, {"at": {13: -1}}, {"at": {12: 0}}):
        refused("QL_E_INVALID", **change)
    for change in ({"at": {12: M + 1}}, {"at": {13: 8}}, {"at": {3: act.arena.size}}, {"at": {8: act.arena.size - 16}}, {"table_off": w.arena.size},
                   {"q_norm_off": w.arena.size}, {"at": {6: act.arena.size}}, {"at": {10: cache.arena.size - 64}}, {"max_pos": 1 << 20}):
        refused("QL_E_RANGE", **change)
    for change in ({"at": {3: args[3] + 4}}, {"at": {6: args[6] + 2}}, {"at": {8: args[8] + 8}}, {"at": {10: args[10] + 4}},
                   {"table_off": args[0].table_off + 4}, {"k_norm_off": args[0].k_norm_off + 8}):
        refused("QL_E_ALIGN", **change)
    for change in ({"at": {8: args[4]}}, {"at": {8: args[3] + 64}}, {"at": {11: args[10]}}, {"at": {8: args[6] // 16 * 16}},
                   {"at": {9: act.arena, 10: args[4] - 2 * KV * D * 4, 12: 6}}):
        refused("QL_E_INVALID", **change)
    with pytest.raises(ql.QlError):
        ctx.rope_table(w.arena, 0, 0, 32, 1e4)
    for bad in ((16, 12, 1e4), (16, 264, 1e4), (16, 32, 0.0), (16, 32, float("inf")), (1 << 20, 32, 1e4)):
        with pytest.raises(ql.QlError):
            ctx.rope_table(w.arena, 0, *bad)
    for change in ({"n_head": 1024}, {"n_kv_head": 4096}):                   # heads of all rows past 2^26
        refused("QL_E_INVALID", at={7: 65535, 12: 1 << 20}, **change)
    ctx.qk_norm_rope(*args)                                                  # the unchanged call runs
    for b in boxes:
        b.release()
