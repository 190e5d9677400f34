"""Batches whose row_start has an entry that it may not have: the sequences on both sides of it have no rows, all others are as ever, in the append and the
attention."""
import numpy as np
import pytest

from tests import test_gpu_paged_append as append
from tests import test_gpu_paged_attention as attention
from tests.paged_ref import Batch

pytestmark = pytest.mark.gpu

FOUR = [(4, 20), (4, 40), (4, 30), (4, 70)]
MANY = [(2, 9 + i % 40) for i in range(150)]                                     # more than a wave looks at at once
CASES = [  # sequences, {entry: what it says}
    (FOUR, {2: -1}), (FOUR, {2: 100}), (FOUR, {2: 2}), (FOUR, {1: 13}), (FOUR, {3: -2**31}), (FOUR, {1: 2**31 - 1, 2: 2**31 - 1}), (FOUR, {0: -3}), (FOUR, {4: 3}),
    (MANY, {10: -1, 67: 1000, 130: 0}), (MANY, {64: 2**31 - 1}), (MANY, {63: -5, 128: 20}),
]


def broken(seqs, changes):
    batch = Batch(seqs, 64, seed=1, pad=3)
    starts = batch.row_start.copy()
    for i, v in changes.items():
        starts[i] = v
    skip = sorted({s for i in changes for s in (i - 1, i) if 0 <= s < len(seqs)})
    for s, (n, L) in enumerate(seqs):                                            # they are none that could have rows, the others are
        r0, r1 = int(starts[s]), int(starts[s + 1])
        assert (0 <= r0 < r1 <= batch.M and r1 - r0 <= min(batch.max_rows, L)) == (s not in skip)
    return batch, starts, skip


@pytest.mark.parametrize("case", range(len(CASES)))
def test_append(ql, ctx, case):
    batch, starts, skip = broken(*CASES[case])
    call = append.Call(ql, ctx, batch, 4, 2, 64, 64, 0, True, case % 2 == 0, False, 0)
    call.box.arena.write(call.box.off("row_start"), starts)
    call.run()
    call.check(skip=skip)
    call.box.release()


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(ql, ctx, case):
    batch, starts, skip = broken(*CASES[case])
    call = attention.Call(ql, ctx, batch, 4, 2, 64, case % 2 == 0, False)
    call.box.arena.write(call.box.off("row_start"), starts)
    call.run()
    call.check(skip=skip)
    call.box.release()
