# SPDX-License-Identifier: MIT
"""Eviction from a paged cache on the GPU, against a plain restatement, bit for bit."""

import math
import random

import pytest
import torch

import beamgrad_amd as bg
from tests import model_reference as ref
from tests import paged_reference as paged

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def problem(dtype, lengths, page, heads, row, layers, joint, seed=0, ties=False):
    g = torch.Generator().manual_seed(seed)
    pages, refs = paged.make_table(paged.sequence_rows(lengths, page), 3, seed)
    pools = [torch.randn(refs.numel(), page, heads, row, generator=g).to(dtype) for _ in range(2 * layers)]
    weights = [torch.randn(len(lengths), 1 if joint else heads, pages.shape[1] * page, generator=g).exp() for _ in range(layers)]
    if ties:
        weights = [w.round() for w in weights]
    return pools, weights, pages, torch.tensor(lengths, dtype=torch.int32), refs


def same_bits(a, b):
    a, b = a.cpu().contiguous(), b.contiguous()
    return a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def check(p, budget, recent=0, first=0, budgets=None):
    pools, weights, pages, lengths, refs = p
    mine = [t.cuda() for t in pools]
    table, got = bg.evict_tokens(mine, [w.cuda() for w in weights], bg.PageTable(pages.cuda(), lengths.cuda(), refs.cuda()),
                                 budget if budgets is None else budgets.cuda(), recent=recent, first=first)
    each = [budget] * len(lengths) if budgets is None else budgets.tolist()
    want = [t.clone() for t in pools]
    new_pages, new_lengths, new_refs, new_weights = ref.evict(want, weights, pages, lengths, refs, each, recent, first)
    assert torch.equal(table.lengths.cpu(), new_lengths)
    assert torch.equal(table.pages.cpu(), new_pages) and torch.equal(table.refs.cpu(), new_refs)
    for i, (a, b) in enumerate(zip(got, new_weights, strict=True)):
        assert same_bits(a, b), i
    for i, (a, b) in enumerate(zip(mine, want, strict=True)):
        assert same_bits(a, b), i
    return table


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("lengths, page, heads, row, layers", [
    ([1], 1, 1, 1, 1), ([40, 0, 17, 100], 16, 2, 8, 2), ([33, 90, 64], 7, 3, 5, 1), ([300], 24, 5, 72, 1), ([70, 65], 8, 1, 33, 3)])
def test_sizes(dtype, joint, lengths, page, heads, row, layers):
    for budget, recent, first in ((0, 0, 0), (1, 0, 0), (16, 4, 2), (40, 40, 3), (64, 100, 100), (29, 0, 29), (60, 7, 0)):
        check(problem(dtype, lengths, page, heads, row, layers, joint, seed=budget), budget, recent, first)


@pytest.mark.parametrize("budget", [1, 1000, 4095, 4096, 5000, 8999])
def test_long_rows(budget):
    """Several rounds of the choice and of the moves."""
    check(problem(torch.bfloat16, [9000, 5000], 16, 2, 8, 1, False, seed=1), budget, budget // 5, 3)


def test_ties_and_strange_weights():
    """Equal weights keep the earlier; infinities, NaN (the least), zeros of both signs, denormals."""
    check(problem(torch.float32, [500, 90], 16, 2, 4, 2, False, ties=True), 77, 5, 2)
    p = problem(torch.float32, [400], 16, 2, 4, 1, False)
    p[1][0].zero_()
    check(p, 100)
    p[1][0][0, 0, ::2] = -0.0
    check(p, 100)
    odd = torch.tensor([math.nan, math.inf, -math.inf, 1e-45, -1e-45, 0.0, -0.0, 3e38, -3e38, 1.0])
    p[1][0].copy_(odd[torch.randint(0, 10, p[1][0].shape, generator=torch.Generator().manual_seed(0))])
    p[1][0][0, 1, ::3] = -math.nan
    for budget in (50, 150, 350, 390):
        check(p, budget, 10, 1)


def test_budgets_of_each_sequence():
    p = problem(torch.float16, [100, 100, 30, 0, 77], 8, 2, 16, 1, False)
    for budgets in (torch.tensor([10, 200, 5, 5, 0], dtype=torch.int32), torch.tensor([2**40, 64, -2**40, 0, 76])):
        check(p, None, 6, 1, budgets=budgets)


def test_sequences_that_stay():
    """Pages that others hold, or that are not there; what is only given back, or kept as
    it is, may be shared."""
    p = problem(torch.float32, [60, 60, 60, 60], 8, 2, 4, 1, False)
    pages, refs = p[2], p[4]
    refs[pages[0, 2].long()] = 2  # written to: sequence 0 stays
    refs[pages[1, 6].long()] = 2  # only given back
    pages[2, 5] = -1  # a token without a page: sequence 2 stays
    refs[pages[3, 0].long()] = 3  # holds the first tokens alone, which stay
    table = check(p, 30, 4, 8)
    assert table.lengths.tolist() == [60, 30, 60, 30]
    p = problem(torch.float32, [64, 8], 8, 1, 4, 1, False)
    p[3][0] = 10**6  # cut to what the table can hold, whose last pages are -1
    assert check(p, 30).lengths[0] == p[2].shape[1] * 8


def test_shared_prompt_pages_are_given_back():
    """Two sequences that hold the same last pages both let them go."""
    p = problem(torch.float32, [64, 64], 8, 1, 4, 1, False)
    pages, refs = p[2], p[4]
    refs[pages[1, 4:8].long()] = 0
    pages[1, 4:8] = pages[0, 4:8]
    refs[pages[0, 4:8].long()] = 2
    table = check(p, 32)
    assert table.lengths.tolist() == [32, 32] and (table.refs[p[2][0, 4:8].long()] == 0).all()


def test_strides_and_many_pools():
    """Pools in turns of one buffer, of several widths, more than one launch holds; weights with strides."""
    S, page, G = 3, 8, 2
    lengths = [50, 33, 70]
    pages, refs = paged.make_table(paged.sequence_rows(lengths, page), 2, 0)
    g = torch.Generator().manual_seed(1)
    base = torch.randn(refs.numel(), page, 80, G, 6, generator=g)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    weights = torch.rand(40, S, G, pages.shape[1] * page, generator=g)
    mine = base.cuda()
    wide = torch.zeros(40, G, S, pages.shape[1] * page + 3, device="cuda")[..., 3:].transpose(1, 2).copy_(weights)
    table, got = bg.evict_tokens(list(mine.unbind(2)), list(wide.unbind(0)), bg.PageTable(pages.cuda(), lengths.cuda(), refs.cuda()), 20,
                                 recent=3, first=1)
    want = [t.clone() for t in base.unbind(2)]
    *_t, new_weights = ref.evict(want, list(weights.unbind(0)), pages, lengths, refs, [20] * S, 3, 1)
    for a, b in zip(mine.unbind(2), want, strict=True):
        assert same_bits(a, b)
    for a, b in zip(got, new_weights, strict=True):
        assert same_bits(a, b)
    p = problem(torch.float32, [40, 50], 8, 2, 4, 1, False)
    p[0].append(torch.randn(p[4].numel(), 8, 2, 3, 5, generator=g).half())  # another width and type
    p[0][1] = torch.randn(p[4].numel(), 8, 2, generator=g)
    check(p, 22, 2)


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("pools_each", [1, 2])
def test_more_sets_of_weights_than_a_launch_holds(pools_each, joint):
    """A model of many layers: two launches choose, and lists of the second are moved by; what stays
    and the pages given back are counted once. Pools of two widths take turns."""
    for sets in (64, 65, 71, 130):
        p = problem(torch.float32, [50, 9, 61, 40, 70], 8, 2, 3, sets, joint, seed=sets)
        pools = p[0][:pools_each * sets]
        pools[1::3] = [t.half() for t in pools[1::3]]
        p = (pools, *p[1:])
        pages, refs = p[2], p[4]
        refs[pages[2, 1].long()] = 2  # written to: sequence 2 stays
        refs[pages[4, 7].long()] = 3  # only given back
        table = check(p, 20, 3, 2)
        assert table.lengths.tolist() == [20, 9, 61, 20, 20]
        # (5 tokens fit a page, so that the second one is not written to)
        assert check(p, None, 3, 2, budgets=torch.tensor([0, 9, 5, 39, 33], dtype=torch.int32)).lengths.tolist() == [0, 9, 5, 39, 33]


def test_evicted_caches_go_on():
    """Evict, extend, write, evict again; the pool's pages come back."""
    p = problem(torch.float32, [120, 90], 8, 2, 4, 1, False)
    pools, weights, pages, lengths, refs = p
    mine, table = [t.cuda() for t in pools], bg.PageTable(pages.cuda(), lengths.cuda(), refs.cuda())
    plain = [t.clone() for t in pools]
    got = [w.cuda() for w in weights]
    for step in range(4):
        table, got = bg.evict_tokens(mine, got, table, 40, recent=8, first=2)
        pages, lengths, refs, weights = ref.evict(plain, weights, pages, lengths, refs, [40, 40], 8, 2)
        counts = torch.tensor([20, 9], dtype=torch.int32)
        table = bg.extend_pages(table, counts.cuda(), 8)
        pages, lengths, refs = paged.extend(pages, lengths, refs, counts, 8)
        news = [torch.randn(2, 20, 2, 4, generator=torch.Generator().manual_seed(step + i)) for i in range(2)]
        bg.write_tokens(mine, [t.cuda() for t in news], table, counts.cuda())
        paged.write(plain, news, pages, lengths, counts)
        fresh = torch.rand(weights[0].shape, generator=torch.Generator().manual_seed(step)) * (weights[0] == 0)
        weights = [weights[0] + fresh]
        got = [got[0] + fresh.cuda()]
        assert torch.equal(table.pages.cpu(), pages) and torch.equal(table.refs.cpu(), refs)
        for a, b in zip(mine, plain, strict=True):
            assert same_bits(a, b)


def test_captured():
    p = problem(torch.bfloat16, [300, 200], 16, 2, 32, 2, False)
    pools, weights = [t.cuda() for t in p[0]], [w.cuda() for w in p[1]]
    table = bg.PageTable(*(t.cuda() for t in p[2:]))

    def step():
        new, w = bg.evict_tokens(pools, weights, table, 100, recent=9, first=1)
        return [*new, *w]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        for w in weights:
            w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(seed)))
        for t, x in zip(pools, p[0], strict=True):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*held, *pools)]
        for t, x in zip(pools, p[0], strict=True):
            t.copy_(x)
        for a, b in zip(got, [*step(), *pools], strict=True):
            assert torch.equal(a, b)


def test_random_calls():
    rng = random.Random(3)
    for seed in range(12):
        lengths = [rng.randrange(0, 200) for _ in range(rng.randrange(1, 6))]
        p = problem(rng.choice(DTYPES), lengths, rng.choice([1, 5, 16, 32]), rng.randrange(1, 4), rng.randrange(1, 20), rng.randrange(1, 3),
                    rng.random() < 0.4, seed, rng.random() < 0.5)
        check(p, rng.randrange(0, 220), rng.randrange(0, 50), rng.randrange(0, 20))
