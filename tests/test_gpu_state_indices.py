# SPDX-License-Identifier: MIT
"""64-bit index tensors with numbers past 32 bits, on the GPU: they count as what
they are, out of range, not as their low words."""

import pytest
import torch

import beamgrad_amd as bg
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

FAR = [2**32, 2**32 + 1, 2**31, 2**40 + 3, -2**31 - 1, -2**32 + 1, 2**63 - 1, -2**63, 2**33 + 2, -2**40]


def low(values):
    """What 32 bits hold of them, at the end of the range that they pass."""
    return torch.tensor([min(max(v, -2**31), 2**31 - 1) for v in values], dtype=torch.int32)


def far(n, start):
    return [FAR[(start + i) % len(FAR)] for i in range(n)]


def cache(S=10, length=20, page=4):
    pages, refs = ref.make_table(ref.sequence_rows([length] * S, page), 60, 1)
    return bg.PageTable(pages.cuda(), torch.full((S,), length, dtype=torch.int32, device="cuda"), refs.cuda())


def test_attention():
    """parents, counts and shared."""
    table, S, N = cache(), 10, 6
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(S, N, 2, 16, device="cuda", generator=g)
    k, v = (torch.randn(table.refs.numel(), 4, 1, 16, device="cuda", generator=g) for _ in range(2))
    parents = torch.tensor([far(N, s) for s in range(S)])
    got = bg.tree_attention(q, k, v, table, parents=parents.cuda())
    assert torch.equal(got, bg.tree_attention(q, k, v, table, parents=torch.full((S, N), -1, device="cuda")))
    counts = far(S, 0)
    got = bg.tree_attention(q, k, v, table, counts=torch.tensor(counts).cuda())
    assert torch.equal(got, bg.tree_attention(q, k, v, table, counts=torch.tensor([N if c > 0 else 0 for c in counts]).cuda()))
    # groups of two: only beams of one group hold the same pages
    pages = table.pages.clone()
    pages[1::2, :4] = pages[::2, :4]
    table = table._replace(pages=pages)
    shared = [2**32 + 3, 12, 2**31, -2**32 + 8, -2**63]
    got = bg.tree_attention(q[:, :1], k, v, table, counts=torch.ones(S, dtype=torch.int32, device="cuda"), beams=2,
                            shared=torch.tensor(shared).cuda())
    assert torch.equal(got, bg.tree_attention(q[:, :1], k, v, table, beams=2, shared=torch.tensor([19, 12, 19, 0, 0]).cuda()))


def test_pages():
    """The counts of extend and write, drafted, keep and kept."""
    table, S = cache(), 10
    for start in range(len(FAR)):
        numbers = [torch.tensor(far(S, start + i)) for i in range(3)]
        narrow = [low(n.tolist()) for n in numbers]
        for a, b in zip(bg.extend_pages(table, numbers[0].cuda(), 4), bg.extend_pages(table, narrow[0].cuda(), 4), strict=True):
            assert torch.equal(a, b)
        news = [torch.randn(S, 3, 5).cuda()]
        pools = [torch.zeros(table.refs.numel(), 4, 5).cuda() for _ in range(2)]
        bg.write_tokens(pools[:1], news, table, numbers[0].cuda())
        bg.write_tokens(pools[1:], news, table, narrow[0].cuda())
        assert torch.equal(*pools)
        eight, two = torch.full((S,), 8, dtype=torch.int32), torch.full((S,), 2, dtype=torch.int32)
        keep = torch.stack([torch.arange(S) % 3, numbers[0]], 1)
        for drafted, keeps, kept in ((numbers[0], two[:, None] + torch.arange(2), two), (eight, keep, two), (eight, keep % 2**31 % 8, numbers[1])):
            wide = torch.randn(table.refs.numel(), 4, 5).cuda()
            pools = [wide, wide.clone()]
            got = bg.keep_tokens(pools[:1], table, drafted.cuda(), keeps.cuda(), kept.cuda())
            want = bg.keep_tokens(pools[1:], table, low(drafted.tolist()).cuda(),
                                  torch.stack([low(row) for row in keeps.tolist()]).cuda(), low(kept.tolist()).cuda())
            assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True)) and torch.equal(*pools)


def test_strides():
    """Index tensors that are not contiguous."""
    table = cache()
    counts = torch.tensor([[3, 2**32], [2**33 + 1, 5]] * 5).cuda()[:, 0]
    got = bg.extend_pages(table, counts, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, bg.extend_pages(table, low(counts.tolist()).cuda(), 4), strict=True))
