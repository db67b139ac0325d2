# SPDX-License-Identifier: MIT
"""Attention over a paged cache on the GPU against 64 bits, at every width and tile of
rows that the kernels lay out in their own way, and where a call has so many items
that each is one workgroup's."""

import math

import pytest
import torch

import beamgrad_amd as bg
from tests import paged_reference as ref
from tests import test_gpu_attention as base

pytestmark = pytest.mark.gpu

F32, F16, BF16 = base.F32, base.F16, base.BF16


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 192, 256, 56, 104, 168, 232])
@pytest.mark.parametrize("N, G", [(10, 1), (7, 4), (15, 4), (50, 2)])
@pytest.mark.parametrize("tree", [False, True])
def test_widths_and_rows(dtype, D, N, G, tree):
    """Tiles of 16, 32, 64 and 128 rows; ragged counts, a cache that several workgroups
    share, and one that holds the asking tokens alone."""
    lengths = [N, N + 60, 700 + N, N + 3]
    base.check(base.build(dtype, lengths, N, G, 1, D, 16, counts=[N, N - 1, N, 1], tree=tree, seed=N + D))


def large(dtype, lengths, counts, N, H, Hkv, D, page, tree, heads, sequences):
    """Against 64 bits on the GPU, for some of the heads and sequences."""
    S = len(lengths)
    g = torch.Generator(device="cuda").manual_seed(0)
    pages, refs = ref.make_table(ref.sequence_rows(lengths, page), 1, 0)
    q = torch.randn(S, N, H, D, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(refs.numel(), page, Hkv, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    parents = None
    if tree:
        at = torch.arange(N)
        parents = (at // 2 + torch.arange(S)[:, None] % 3 - 1).clamp(max=N).int()
        parents[:, 0] = -1
    table = bg.PageTable(pages.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), refs.cuda())
    out, lse = bg.tree_attention(q, k, v, table, counts=torch.tensor(counts).cuda(), parents=None if parents is None else parents.cuda(),
                                 return_lse=True)
    for s in sequences:
        n, c = lengths[s], counts[s]
        assert bool((out[s, c:] == 0).all()) and bool(torch.isneginf(lse[s, c:]).all())
        if c == 0:
            continue
        held = pages[s, :-(-n // page)].long().cuda()
        seen = torch.ones(c, n, dtype=torch.bool)
        seen[:, n - c:] = False
        for i in range(c):
            seen[i, [n - c + j for j in ref.seen_by(i, c, None if parents is None else parents[s])]] = True
        seen = seen.cuda()
        for h in heads:
            key, value = (t[held, :, h // (H // Hkv)].flatten(0, 1)[:n].double() for t in (k, v))
            row = q[s, :c, h].double()
            score = (row @ key.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
            p = torch.softmax(score, -1)
            error = (row.abs() @ key.abs().T).amax(-1) / math.sqrt(D) * (D + 2) * 2.0**-24
            want = (p @ value, torch.logsumexp(score, -1), p @ value.abs(), error)
            bound, lse_bound = ref.attention_bounds(dtype, *want, n, 8.0)
            assert bool(((out[s, :c, h].double() - want[0]).abs() <= bound).all()), (s, h)
            assert bool(((lse[s, :c, h].double() - want[1]).abs() <= lse_bound).all()), (s, h)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_whole_items_of_few_sequences(dtype):
    """1024 items, two for each of 512 workgroups: the entries are sorted by their
    keys."""
    N, H = 2048, 32
    large(dtype, [N + 70, N - 100], [N, N - 100], N, H, H, 32, 32, False, range(0, H, 7), range(2))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_whole_items_of_many_sequences(dtype, D):
    """More entries than the workgroup that sorts them has threads."""
    S, N, H = 150, 256, 4
    lengths = [N + (s * 37) % 100 for s in range(S)]
    counts = [N - (s % 5) * 30 for s in range(S)]
    lengths[3], counts[3], lengths[77], counts[77] = 0, 0, 5, 5
    large(dtype, lengths, counts, N, H, H, D, 16, False, (0, 3), (0, 1, 3, 4, 76, 77, 149))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_whole_items_of_trees(dtype):
    S, N, H = 18, 130, 32
    lengths = [N + 40 + (s * 11) % 50 for s in range(S)]
    large(dtype, lengths, [N - s for s in range(S)], N, H, H, 64, 16, True, (0, 17, 31), (0, 5, 17))
