"""GPU: cache rows moved (ql_kv_move). Copies: every result is bit-exact."""
import numpy as np
import pytest

from tests.arena_box import Box

pytestmark = pytest.mark.gpu


def regions(ql, ctx, count, T, row_bytes, seed, gap=0):
    g = np.random.default_rng(seed)
    b = Box(ql, ctx)
    offs = [b.put(i, g.integers(0, 2**32, (T, row_bytes // 4), dtype=np.uint32), align=16, gap=16 * gap) for i in range(count)]
    b.place()
    return b, offs


def moved(dst, src, dst_row, src_row, n, rows=None):
    out = [d.copy() for d in dst]
    for o, s in zip(out, src):
        for i in range(n):
            at = i if rows is None else int(rows[i])
            if at >= 0 and src_row + at < len(s):
                o[dst_row + i] = s[src_row + at]
    return out


def same(b, want):
    for i, w in enumerate(want):
        assert np.array_equal(b.get(i), w), i


@pytest.mark.parametrize("count,T,row_bytes,n", [(1, 1, 16, 1), (2, 9, 48, 7), (48, 40, 512, 33), (56, 70, 2048, 70), (130, 5, 32, 4), (256, 3, 16, 2),
                                                 (3, 2000, 1040, 1999)])
def test_copy_to_another_cache(ql, ctx, count, T, row_bytes, n):
    a, ao = regions(ql, ctx, count, T, row_bytes, 1)
    b, bo = regions(ql, ctx, count, T + 3, row_bytes, 2, gap=1)
    dst_row, src_row = 2, T - n
    want = moved([b.get(i) for i in range(count)], [a.get(i) for i in range(count)], dst_row, src_row, n)
    ctx.kv_move(b.arena, bo, T + 3, a.arena, ao, T, row_bytes, dst_row, src_row, n)
    same(b, want)
    a.release()
    b.release()


@pytest.mark.parametrize("n", [1, 4, 8, 33, 160, 256])
@pytest.mark.parametrize("row_bytes", [16, 256, 1008, 2048])
@pytest.mark.parametrize("order", ["ascending", "any", "twice", "reversed"])
def test_gather_in_place(ql, ctx, n, row_bytes, order):
    """A list over the region itself: as if all rows were read before any is written."""
    T, past, count = 400, 100, 5
    g = np.random.default_rng(n)
    rows = {"ascending": np.sort(g.permutation(300)[:n]), "any": g.permutation(300)[:n], "twice": g.integers(0, max(2, n // 2), n),
            "reversed": np.arange(n)[::-1]}[order].astype(np.int32)
    a, ao = regions(ql, ctx, count, T, row_bytes, 3)
    act = Box(ql, ctx)
    act.put("rows", rows, gap=4)
    act.place()
    start = [a.get(i) for i in range(count)]
    ctx.kv_move(a.arena, ao, T, a.arena, ao, T, row_bytes, past, past, n, act.arena, act.off("rows"))
    same(a, moved(start, start, past, past, n, rows))
    # without a list, shifted by one row onto itself
    if n < 256:
        start = [a.get(i) for i in range(count)]
        ctx.kv_move(a.arena, ao, T, a.arena, ao, T, row_bytes, past + 1, past, n)
        same(a, moved(start, start, past + 1, past, n))
    a.release()
    act.release()


def test_bad_entries_leave_their_rows(ql, ctx):
    T, row_bytes, count = 20, 64, 3
    rows = np.array([3, -1, 2**31 - 1, 12, 13, -2**31, 0, 12], np.int32)
    for other in (False, True):
        a, ao = regions(ql, ctx, count, T, row_bytes, 4)
        b, bo = regions(ql, ctx, count, T, row_bytes, 5) if other else (a, ao)
        act = Box(ql, ctx)
        act.put("rows", rows)
        act.place()
        start, src = [b.get(i) for i in range(count)], [a.get(i) for i in range(count)]
        ctx.kv_move(b.arena, bo, T, a.arena, ao, T, row_bytes, 8, 7, len(rows), act.arena, act.off("rows"))
        same(b, moved(start, src, 8, 7, len(rows), rows))
        for x in {a, b}:
            x.release()
        act.release()


def test_gather_from_another_cache_of_any_length(ql, ctx):
    T, row_bytes, n, count = 3000, 96, 2500, 3
    rows = np.random.default_rng(7).integers(0, T, n).astype(np.int32)
    a, ao = regions(ql, ctx, count, T, row_bytes, 8)
    b, bo = regions(ql, ctx, count, n + 1, row_bytes, 9)
    act = Box(ql, ctx)
    act.put("rows", rows)
    act.place()
    want = moved([b.get(i) for i in range(count)], [a.get(i) for i in range(count)], 1, 0, n, rows)
    ctx.kv_move(b.arena, bo, n + 1, a.arena, ao, T, row_bytes, 1, 0, n, act.arena, act.off("rows"))
    same(b, want)
    for x in (a, b, act):
        x.release()


def test_offsets_past_32_bits(ql, ctx):
    """The last rows of a 4.5 GiB region to its own beginning, and back."""
    row_bytes = 4096
    T = (9 << 29) // row_bytes
    a = ctx.arena(T * row_bytes)
    tail = np.random.default_rng(1).integers(0, 2**32, (6, row_bytes // 4), dtype=np.uint32)
    a.write((T - 6) * row_bytes, tail)
    ctx.kv_move(a, [0], T, a, [0], T, row_bytes, 1, T - 6, 6)
    assert np.array_equal(a.read(row_bytes, tail.shape, np.uint32), tail)
    b = Box(ql, ctx)
    b.put("rows", np.array([5, 0, 3], np.int32))
    b.place()
    ctx.kv_move(a, [0], T, a, [0], T, row_bytes, T - 3, T - 6, 3, b.arena, b.off("rows"))
    assert np.array_equal(a.read((T - 3) * row_bytes, (3, row_bytes // 4), np.uint32), tail[[5, 0, 3]])
    a.release()
    b.release()


def test_refusals(ql, ctx):
    T, rb = 16, 64
    a, ao = regions(ql, ctx, 2, T, rb, 1)
    b, bo = regions(ql, ctx, 2, T, rb, 2)
    act = Box(ql, ctx)
    act.put("rows", np.arange(16, dtype=np.int32))
    act.place()
    before = [b.get(i) for i in range(2)]

    def refused(name, *args):
        with pytest.raises(ql.QlError) as e:
            ctx.kv_move(*args)
        assert e.value.name == name, (args, e.value)

    A, B = a.arena, b.arena
    refused("QL_E_INVALID", B, [], T, A, [], T, rb, 0, 0, 1)
    refused("QL_E_INVALID", B, bo * 129, T, A, ao * 129, T, rb, 0, 0, 1)
    for bad in (0, 8, 24, -16):
        refused("QL_E_INVALID", B, bo, T, A, ao, T, bad, 0, 0, 1)
    refused("QL_E_INVALID", B, bo, T, A, ao, T, rb, -1, 0, 1)
    refused("QL_E_INVALID", B, bo, T, A, ao, T, rb, 0, -1, 1)
    refused("QL_E_INVALID", B, bo, T, A, ao, T, rb, 0, 0, -1)
    refused("QL_E_RANGE", B, bo, T, A, ao, T, rb, 1, 0, T)
    refused("QL_E_RANGE", B, bo, T, A, ao, T, rb, 0, 1, T)
    refused("QL_E_RANGE", B, bo, T, A, [ao[0], A.size], T, rb, 0, 0, 1)
    refused("QL_E_RANGE", B, [bo[0], B.size - rb], T, A, ao, T, rb, 0, 0, 1)
    refused("QL_E_ALIGN", B, [bo[0] + 8, bo[1]], T, A, ao, T, rb, 0, 0, 1)
    refused("QL_E_RANGE", B, bo, T, A, ao, T, rb, 0, 0, 4, act.arena, act.arena.size - 8)
    refused("QL_E_ALIGN", B, bo, T, A, ao, T, rb, 0, 0, 4, act.arena, act.off("rows") + 2)
    refused("QL_E_INVALID", B, [bo[0], bo[0] + 2 * rb], 8, A, ao, T, rb, 0, 0, 4)              # two written regions meet
    refused("QL_E_INVALID", A, [ao[0], ao[0] + rb], 8, A, ao, T, rb, 0, 0, 4)                  # onto another region's source
    refused("QL_E_INVALID", A, [ao[0] + 16], 8, A, [ao[0]], 8, rb, 0, 0, 4)                    # partly onto itself
    refused("QL_E_INVALID", B, bo, T, A, ao, T, rb, 0, 0, 4, B, bo[0] + rb)                    # onto the list
    big, go = regions(ql, ctx, 1, 600, 16, 3)
    refused("QL_E_INVALID", big.arena, go, 600, big.arena, go, 600, 16, 1, 0, 257)             # onto itself, too long
    ctx.kv_move(big.arena, go, 600, big.arena, go, 600, 16, 300, 0, 300)                       # apart in one region: any length
    with pytest.raises(ValueError):
        ctx.kv_move(B, bo, T, A, ao[:1], T, rb, 0, 0, 1)
    ctx.kv_move(B, bo, T, A, ao, T, rb, 0, 0, 0)                                               # nothing to do
    same(b, before)
    for x in (a, b, act, big):
        x.release()
