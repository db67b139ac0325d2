# SPDX-License-Identifier: MIT
"""Beams over shared pages on the GPU against 64 bits: at every width, with a few
and with many rows each, and in more groups than one launch takes."""

import math

import pytest
import torch

from tests import paged_reference as ref
from tests import test_gpu_attention as base

pytestmark = pytest.mark.gpu

F32, F16, BF16 = base.F32, base.F16, base.BF16


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 72, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("K, N, G, tree", [(3, 1, 4, False), (3, 5, 4, True), (5, 7, 4, False), (4, 9, 5, True)])
def test_widths(dtype, D, K, N, G, tree):
    """Tiles of 16 to 128 rows that several beams share, one after the other."""
    shared = [64, 33]
    lengths = [shared[s // K] + N + (5 * s) % 37 for s in range(2 * K)]
    counts = [N if s % 3 else max(N - 2, 0) for s in range(2 * K)]
    base.check(base.build(dtype, lengths, N, G, 1, D, 16, K=K, shared=shared, counts=counts, tree=tree, seed=K))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("K, N, G, D", [(2, 16, 8, 64), (4, 28, 4, 64), (3, 33, 2, 128), (2, 140, 1, 72), (5, 61, 1, 128)])
@pytest.mark.parametrize("tree", [False, True])
def test_many_rows_a_beam(dtype, K, N, G, D, tree):
    """Beams that fill tiles by themselves, and others that nearly do."""
    shared = [80, 20]
    lengths = [shared[s // K] + N + (7 * s) % 23 for s in range(2 * K)]
    base.check(base.build(dtype, lengths, N, G, 1, D, 16, K=K, shared=shared, tree=tree, seed=N))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N", [6, 40])
def test_unseen_values_beside_shared_pages(dtype, N):
    """An infinite value in a drafted token of one beam reaches the rows that see it,
    and no other row or beam."""
    K, prefix = 2, 300
    c = base.build(dtype, [prefix + N] * K, N, 2, 1, 64, 16, K=K, shared=[prefix], tree=True, seed=N)
    want = base.expected(c)
    at = prefix + 3
    c["v"][int(c["pages"][0, at // 16]), at % 16, 0, 7] = math.inf
    out, lse = (t.cpu().double() for t in base.run(c))
    bound, lse_bound = ref.attention_bounds(dtype, *want, prefix + N, 8.0)
    for s in range(K):
        for i in range(N):
            if s == 0 and 3 in ref.seen_by(i, N, c["parents"][s]):
                assert bool(torch.isinf(out[s, i, :, 7]).all()) and bool(out[s, i, :, :7].isfinite().all())
            else:
                assert bool(((out[s, i] - want[0][s, i]).abs() <= bound[s, i]).all())
    assert bool(((lse - want[1]).abs() <= lse_bound).all())


def test_groups_of_several_launches():
    """More partial results than a launch keeps: 60 groups of four beams with 64 heads
    of float32, 200 wide, are two launches."""
    K, groups, H, D = 4, 60, 64, 200
    shared = [(3 * b) % 11 for b in range(groups)]
    lengths = [shared[s // K] + 1 + s % 4 for s in range(groups * K)]
    c = base.build(F32, lengths, 1, H, H, D, 4, K=K, shared=shared)
    base.check(c)
