"""Host only: masks and depths of a drafted tree (ql_tree_masks), and refusals that need no device."""
import ctypes

import numpy as np
import pytest


def plain(parents):
    M = len(parents)
    seen, depth = np.zeros((M, M), bool), []
    for m in range(M):
        j, d = m, -1
        while j >= 0:
            seen[m, j] = True
            j, d = parents[j], d + 1
        depth.append(d)
    words = np.zeros((M, (M + 63) // 64), np.uint64)
    for m, j in np.argwhere(seen):
        words[m, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return words, depth


@pytest.mark.parametrize("M", [1, 2, 7, 63, 64, 65, 128, 129, 256])
def test_masks_and_depths(ql, M):
    g = np.random.default_rng(M)
    for parents in (np.arange(-1, M - 1), np.full(M, -1), np.array([int(g.integers(-1, m)) if m else -1 for m in range(M)])):
        masks, depths = ql.tree_masks(parents)
        words, depth = plain(list(parents))
        assert np.array_equal(masks, words) and np.array_equal(depths, depth)


def test_bad_trees(ql):
    for parents in ([0], [-1, 1], [-1, 2, 0], [-2], [-1, 0, -5], [], [-1] * 257):
        with pytest.raises(ql.QlError) as e:
            ql.tree_masks(parents)
        assert e.value.name == "QL_E_INVALID"


def test_either_result_may_be_left_out(ql):
    L, p = ql.lib(), np.array([-1, 0, 0], np.int32)
    d, m = np.zeros(3, np.int32), np.zeros(3, np.uint64)
    assert L.ql_tree_masks(3, p.ctypes.data, None, d.ctypes.data) == 0 and list(d) == [0, 1, 1]
    assert L.ql_tree_masks(3, p.ctypes.data, m.ctypes.data, None) == 0 and list(m) == [1, 3, 5]
    assert L.ql_tree_masks(3, None, m.ctypes.data, None) == -10


def test_null_handles(ql):
    L, none = ql.lib(), ql.QL_NONE
    assert L.ql_rope_table(None, None, 0, 1, 8, 1e4) == -10
    assert L.ql_qk_norm_rope(None, None, None, None, 0, 0, 0, 0, 1, 0, None, 0, 0, 1, 0) == -10
    assert L.ql_attention_tree(None, None, 0, None, 0, 0, 0, 1, 1, 1, 1, 8, 0, none, 0) == -10
    assert L.ql_token_logprobs(None, None, 0, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0) == -10
    assert L.ql_kv_move(None, None, None, 1, None, None, 1, 1, 16, 0, 0, 1, None, none) == -10
    assert ctypes.sizeof(ql.RopeDesc) == 3 * 8 + 12 * 4


def test_parents_past_32_bits(ql):
    for parents in (np.array([-1, 2**32 - 1]), np.array([-1, 2**32]), np.array([-(2**40), 0])):
        with pytest.raises(ql.QlError):
            ql.tree_masks(parents)


def test_parents_that_are_no_rows(ql):
    """Fractions and NaN, which a cast would make row 0 or -1 of; whole numbers in any type are rows."""
    for parents in ([-1, 0.7], [-1, -0.5], [-1, 0, float("nan")], [-1, float("inf")], np.array([-1, 0, 0.999], np.float32)):
        with pytest.raises(ql.QlError) as e:
            ql.tree_masks(parents)
        assert e.value.name == "QL_E_INVALID"
    for parents in ([-1.0, 0.0, 1.0], np.array([-1, 0, 1], np.int64), np.array([-1, 0, 1], np.int8), (-1, 0, 1)):
        masks, depths = ql.tree_masks(parents)
        assert [int(w) for w in masks[:, 0]] == [1, 3, 7] and list(depths) == [0, 1, 2]


def test_plans_of_tree_attention(ql):
    """ql_plan_attention_tree (host only): the GPU tests' instances, ranges that cover the keys, the call's refusals."""
    from tests.test_gpu_attn_tree import PLANS, SHAPES

    for M, H, KV, D, past, half, want, label in PLANS:
        p = ql.plan_attention_tree(int(half), past + M, M, H, KV, D, past)
        assert (p.pairs, p.waves, p.nsplit) == want, label
    seen = set()
    for M, H, KV, D, past, label in SHAPES:
        for half in (0, 1):
            p = ql.plan_attention_tree(half, past + M, M, H, KV, D, past)
            seen.add((p.pairs, p.waves))
            assert p.nsplit * p.keys_per_split >= past + M and p.workgroups * p.pairs >= M * H * p.nsplit, label
    assert seen == {(1, 1), (16, 4), (16, 8)}
    for bad in ((2, 64, 4, 4, 2, 64, 10), (0, 13, 4, 4, 2, 64, 10), (0, 64, 0, 4, 2, 64, 10), (0, 64, 257, 4, 2, 64, 10), (0, 64, 4, 4, 3, 64, 10),
                (0, 64, 4, 4, 2, 68, 10), (0, 64, 4, 4, 2, 264, 10), (0, 64, 4, 4, 2, 64, -1), (0, 2**31 - 1, 4, 4, 2, 64, 2**30 + 1)):
        with pytest.raises(ql.QlError):
            ql.plan_attention_tree(*bad)
    assert ql.lib().ql_plan_attention_tree(0, 64, 4, 4, 2, 64, 10, None) == -10


def test_rows_at_once_are_the_formula(ql):
    """The GPU tests' two forms of the formula agree, with rows that see nothing, NaN and infinities in seen and unseen keys."""
    from tests.test_gpu_attn_tree import formula, many, seen_of, tree

    g, M, past = np.random.default_rng(1), 9, 20
    masks, _ = ql.tree_masks(tree(M, 2))
    masks[4] = 0
    for p in (0, past):
        for what, value in ((None, 0), ("k", np.nan), ("k", np.inf), ("k", -np.inf), ("v", np.nan), ("v", np.inf), ("v", -np.inf)):
            q, k, v = (g.standard_normal(s).astype(np.float32) for s in ((M, 4, 8), (p + M, 2, 8), (p + M, 2, 8)))
            if what:
                (k if what == "k" else v)[[p + 3, p + M - 1], :, 5] = value
            a, b = formula(q, k, v, seen_of(masks, M, p)), many(q, k, v, seen_of(masks, M, p))
            assert np.allclose(a[0], b[0], rtol=1e-12, atol=1e-12, equal_nan=True)
            at = np.isfinite(a[0]) & (a[0] != 0)
            assert np.allclose(a[1][at], b[1][at], rtol=1e-9)
