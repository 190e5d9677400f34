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
