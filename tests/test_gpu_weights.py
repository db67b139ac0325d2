# SPDX-License-Identifier: MIT
"""The attention that cached tokens get, on the GPU, against a 64-bit restatement."""

import math
import random

import pytest
import torch

import beamgrad_amd as bg
from tests import model_reference as ref
from tests import paged_reference as paged

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def problem(dtype, S, N, H, Hkv, D, page, lengths, counts=None, tree=False, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    pages, refs = paged.make_table(paged.sequence_rows(lengths, page), 3, seed)
    q = (torch.randn(S, N, H, D, generator=g) * spread).to(dtype)
    k = torch.randn(refs.numel(), page, Hkv, D, generator=g).to(dtype)
    weights = torch.rand(S, Hkv, pages.shape[1] * page, generator=g)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    rng = random.Random(seed)
    parents = torch.tensor([[rng.randrange(-1, i) if i else -1 for i in range(N)] for _ in range(S)], dtype=torch.int32) if tree else None
    counts = torch.tensor(counts, dtype=torch.int32) if counts is not None else None
    return dict(q=q, k=k, weights=weights, table=(pages, lengths, refs), parents=parents, counts=counts, scale=1.0 / math.sqrt(D))


def check(p, lse=None, index=lambda t: t, atol=0.0):
    S, N = p["q"].shape[:2]
    pages, lengths, refs = p["table"]
    counts = p["counts"] if p["counts"] is not None else torch.full((S,), N)
    table = bg.PageTable(pages.cuda(), lengths.cuda(), refs.cuda())
    more = {n: None if p[n] is None else index(p[n]).cuda() for n in ("parents", "counts")}
    q, k = p["q"].cuda(), p["k"].cuda()
    if lse is None:
        _out, lse = bg.tree_attention(q, k, k, table, return_lse=True, scale=p["scale"], **more)
    weights = p["weights"].cuda()
    bg.accumulate_weights(weights, q, k, lse.cuda(), table, scale=p["scale"], **more)
    want, bound = ref.accumulate(p["weights"], p["q"], p["k"], lse.cpu(), pages, lengths, counts, p["parents"], p["scale"])
    far = (weights.cpu().double() - want).abs() - bound - atol
    assert far.max() <= 0, (float(far.max()), far.argmax())
    # what is no asked-for token's place keeps its bits
    still = bound == 0
    assert torch.equal(weights.cpu()[still], p["weights"][still])
    return weights


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 64, 72, 128, 136, 192, 200, 256])
def test_widths(dtype, D):
    check(problem(dtype, 2, 3, 4, 2, D, 16, [70, 300]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [40, 64, 128, 192, 256])
@pytest.mark.parametrize("N", [4, 8, 14, 30, 45, 60, 80, 96, 100])
def test_rows_of_every_number(dtype, D, N):
    """One block of rows, as many as pass keys' way holds, and more; trees and chains."""
    lengths, counts = [130 + N, N, 700, 3], [N, N, N - 3, 2]
    check(problem(dtype, 4, N, 8, 2, D, 24, lengths, counts, tree=True, seed=N))
    check(problem(dtype, 4, N, 8, 2, D, 24, lengths, counts, seed=N))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths, counts, N, H, Hkv, page", [
    ([1], None, 1, 1, 1, 1),
    ([1, 700, 63, 64, 65], None, 1, 8, 2, 16),
    ([40, 0, 9, 30], [1, 0, 5, 3], 5, 6, 3, 7),
    ([257, 256, 255], [20, 1, 17], 20, 5, 1, 24),
    ([30, 31], None, 30, 3, 3, 16),
    ([2000], None, 90, 16, 1, 64),
    ([12, 5], [99, -4], 10, 2, 1, 8),
])
def test_lengths_and_counts(dtype, lengths, counts, N, H, Hkv, page):
    check(problem(dtype, len(lengths), N, H, Hkv, 64, page, lengths, counts))
    check(problem(dtype, len(lengths), N, H, Hkv, 64, page, lengths, counts, tree=True, seed=1), index=lambda t: t.long())


def test_many_rows_over_few_keys():
    """Rows that are split, so that their sums are joined; odd numbers of blocks."""
    p = problem(torch.bfloat16, 2, 500, 6, 2, 64, 16, [530, 517], [500, 333])
    size = p["table"][0].shape
    assert size[1] * 16 < 1000
    check(p)
    check(problem(torch.float32, 1, 130, 16, 1, 128, 16, [140]))


def test_a_long_cache_and_many_sequences():
    check(problem(torch.float16, 3, 1, 4, 2, 64, 128, [5000, 1, 2111]))
    rng = random.Random(0)
    check(problem(torch.bfloat16, 300, 1, 2, 1, 16, 4, [rng.randrange(0, 30) for _ in range(300)]))
    check(problem(torch.bfloat16, 300, 6, 2, 1, 16, 4, [rng.randrange(0, 60) for _ in range(300)]))


def test_large_trees():
    p = problem(torch.bfloat16, 2, 512, 2, 1, 32, 32, [900, 512], tree=True)
    p["parents"][0, ::7] = 600  # no earlier node
    p["parents"][1] = torch.arange(-1, 511)  # a chain
    check(p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [4, 32, 80, 256])
def test_bad_pages_masks_and_empty_rows(dtype, H):
    """Pages that are not there, lengths past the table, NaN behind a sequence and in
    unseen places, rows whose log-sum is -inf."""
    p = problem(dtype, 4, 4, H, 2, 64, 8, [40, 33, 20, 8], [4, 2, 4, 3])
    pages, lengths, refs = p["table"]
    nan_pages = [int(pages[1, 4]), int(pages[3, 0])]
    pages[0, 1], pages[0, 2] = -7, refs.numel()
    lengths[2] = 10**6  # cut to what the table holds; its last pages are -1
    p["k"][nan_pages[0], 1:] = math.nan  # behind token 32 of sequence 1
    p["q"][1, 2:] = math.nan  # tokens that do not ask
    p["q"][3, 3] = math.inf
    check(p)
    # no page at all: every row is empty
    pages[3] = -1
    lse = torch.randn(4, 4, H).abs() + 5
    lse[3] = -math.inf
    lse[0, 0] = -math.inf
    lse[0, 1, 2] = math.inf
    check(p, lse)


def test_places_of_the_attention_add_to_one():
    """Every asking row gives a weight of one altogether."""
    p = problem(torch.float32, 3, 7, 8, 4, 64, 16, [300, 45, 7])
    p["weights"].zero_()
    got = check(p)
    assert ((got.sum(-1) - 7 * 2).abs() <= 7 * 2 * 400 * ref.STEP).all()


def test_strides_of_weights_queries_and_cache():
    p = problem(torch.bfloat16, 2, 3, 4, 2, 64, 16, [70, 300])
    pages, lengths, refs = (t.cuda() for t in p["table"])
    table = bg.PageTable(pages, lengths, refs)
    q, k = p["q"].cuda(), p["k"].cuda()
    lse = bg.tree_attention(q, k, k, table, return_lse=True)[1]
    want = p["weights"].cuda()
    bg.accumulate_weights(want, q, k, lse, table)
    places = want.shape[2]
    wide = torch.zeros(2, 2, places + 5, device="cuda")[..., :places].copy_(p["weights"])
    turned = torch.zeros(2, 2, places, device="cuda").transpose(0, 1).copy_(p["weights"])
    far_q = torch.zeros(2, 5, 6, 80, device="cuda", dtype=torch.bfloat16)[:, 1:4, 1:5, 8:72].copy_(q)
    odd_q = torch.zeros(2, 3, 4, 67, device="cuda", dtype=torch.bfloat16)[..., 3:].copy_(q)
    far_k = torch.zeros(k.shape[0], 2, 16, 3, 64, device="cuda", dtype=torch.bfloat16)[:, 1, :, :2].copy_(k)
    for w in (wide, turned):
        for a in (far_q, odd_q):
            w.copy_(p["weights"])
            bg.accumulate_weights(w, a, far_k, lse.transpose(0, 1).contiguous().transpose(0, 1), table)
            assert torch.equal(w, want)


def test_memory_that_meets_is_refused():
    """Weights in a part of the queries, keys or log-sums; between two of the cache's rows they fit."""
    table = bg.PageTable(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1,), 4, dtype=torch.int32, device="cuda"),
                         torch.ones(1, dtype=torch.int32, device="cuda"))
    buffer = torch.zeros(1 << 10, device="cuda")
    q, lse, k = buffer[:16].view(1, 1, 2, 8), buffer[64:66].view(1, 1, 2), buffer[128:192].view(1, 4, 1, 16)[..., :8]
    for at in (8, 62, 130):
        with pytest.raises(ValueError, match="share no memory"):
            bg.accumulate_weights(buffer[at:at + 4].view(1, 1, 4), q, k, lse, table)
    weights = buffer[136:140].view(1, 1, 4)
    bg.accumulate_weights(weights, q, k, lse, table)
    assert torch.equal(weights.cpu(), torch.tensor([[[2.0, 2.0, 2.0, 2.0]]]))  # e^(0 - 0), of two heads


def test_the_same_every_time_and_captured():
    p = problem(torch.bfloat16, 2, 300, 4, 2, 64, 16, [400, 333])
    pages, lengths, refs = (t.cuda() for t in p["table"])
    table = bg.PageTable(pages, lengths, refs)
    q, k = p["q"].cuda(), p["k"].cuda()
    lse = bg.tree_attention(q, k, k, table, return_lse=True)[1]
    weights = p["weights"].cuda()

    def step():
        bg.accumulate_weights(weights, q, k, lse, table)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        start = torch.rand(weights.shape, generator=torch.Generator().manual_seed(seed))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        weights.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        got = weights.clone()
        weights.copy_(start)
        step()
        assert torch.equal(got, weights)


def test_weights_noticed_as_written():
    p = problem(torch.float32, 1, 1, 1, 1, 8, 4, [5])
    weights = p["weights"].cuda()
    version = weights._version
    table = bg.PageTable(*(t.cuda() for t in p["table"]))
    bg.accumulate_weights(weights, p["q"].cuda(), p["k"].cuda(), torch.zeros(1, 1, 1, device="cuda"), table)
    assert weights._version > version
