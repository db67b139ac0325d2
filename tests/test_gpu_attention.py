# SPDX-License-Identifier: MIT
"""Attention over a paged cache on the GPU against 64 bits, at the sizes, masks
and layouts where it can go wrong."""

import math

import pytest
import torch

import beamgrad_amd as bg
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def build(dtype, lengths, N, H, Hkv, D, page, *, K=1, shared=None, counts=None, tree=False, seed=0, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    S = len(lengths)
    rows = ref.sequence_rows(lengths, page, shared, K)
    pages, refs = ref.make_table(rows, 3, seed)
    n = refs.numel()
    q = (torch.randn(S, N, H, D, generator=g) * spread).to(dtype)
    k, v = (torch.randn(n, page, Hkv, D, generator=g).to(dtype) for _ in range(2))
    # places that hold no token must not matter
    held = torch.zeros(n, page, dtype=torch.bool)
    for s, length in enumerate(lengths):
        for t in range(length):
            held[pages[s, t // page], t % page] = True
    k[~held], v[~held] = math.nan, math.inf
    parents = None
    if tree:
        parents = torch.full((S, N), -1, dtype=torch.int32)
        for s in range(S):
            for i in range(1, N):
                parents[s, i] = int(torch.randint(-1, i, (1,), generator=g))
    counts = [min(N, x) for x in lengths] if counts is None else counts
    return dict(q=q, k=k, v=v, pages=pages, lengths=torch.tensor(lengths, dtype=torch.int32), refs=refs,
                counts=torch.tensor(counts, dtype=torch.int32), parents=parents, K=K,
                shared=None if shared is None else torch.tensor(shared, dtype=torch.int32))


def run(c, lse=True, scale=None, **more):
    cu = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    cu.update(more)
    return bg.tree_attention(cu["q"], cu["k"], cu["v"], bg.PageTable(cu["pages"], cu["lengths"], cu["refs"]),
                             parents=cu["parents"], counts=cu["counts"], beams=c["K"], shared=cu["shared"], scale=scale,
                             return_lse=lse)


def expected(c, scale=None):
    scale = 1.0 / math.sqrt(c["q"].shape[-1]) if scale is None else scale
    return ref.attention(c["q"], c["k"], c["v"], c["pages"], c["lengths"], c["counts"], c["parents"], scale)


def check(c, got=None, scale=None, want=None):
    out, lse = run(c, scale=scale) if got is None else got
    want = expected(c, scale) if want is None else want
    top = c["v"].float().nan_to_num(0, 0, 0).abs().max().item()
    bound, lse_bound = ref.attention_bounds(c["q"].dtype, *want, int(c["lengths"].max()), top)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want[1]))
    live = ~torch.isneginf(lse)
    off = (out - want[0]).abs()
    assert bool((off <= bound).all()), f"out is off by {(off / bound.clamp(min=1e-300)).max():.3g} times its bound"
    assert bool((out[~live] == 0).all())
    off = (lse - want[1])[live].abs()
    assert bool((off <= lse_bound[live]).all()), f"lse is off by {off.max():.3g}"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [8, 64, 72, 128, 136, 200, 256])
def test_widths(dtype, D):
    """One token a sequence: every padded width, lengths of zero and one."""
    check(build(dtype, [0, 1, 17, 33, 200], 1, 6, 2, D, 16))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N, H, Hkv", [(1, 1, 1), (1, 8, 8), (1, 24, 2), (5, 4, 1), (7, 15, 5), (33, 2, 2), (64, 6, 3), (150, 2, 1)])
def test_chains(dtype, N, H, Hkv):
    """The end of a prompt: every tile of rows, counts below N and of zero."""
    lengths = [N, N + 1, 3, N + 90]
    check(build(dtype, lengths, N, H, Hkv, 64, 24, counts=[N, max(N // 2, 1), 0, min(N, 60)], seed=N))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N, G, D", [(2, 1, 64), (7, 3, 72), (33, 4, 128), (61, 4, 64), (100, 1, 256), (130, 2, 192)])
def test_trees(dtype, N, G, D):
    lengths = [N, N + 40, N + 5, 200 + N]
    check(build(dtype, lengths, N, 2 * G, 2, D, 16, counts=[N, 1, N - 1, N], tree=True, seed=N))


def test_the_largest_tree():
    check(build(F16, [512 + 9], 512, 1, 1, 32, 20, tree=True))


def test_parents_that_are_no_earlier_token():
    c = build(F32, [30, 31], 6, 2, 1, 32, 8, tree=True)
    c["parents"][0] = torch.tensor([5, 1, 7, 2, -9, 100000], dtype=torch.int32)
    c["parents"][1] = torch.tensor([0, 0, 2, 2**31 - 1, -2**31, 4], dtype=torch.int32)
    check(c)
    check(c, run(c, parents=c["parents"].long().cuda(), counts=c["counts"].long().cuda()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K, G, page, shared", [(2, 1, 16, [40, 0]), (4, 4, 16, [64, 7]), (8, 4, 24, [150, 100]), (16, 12, 8, [33, 200]), (3, 5, 1, [9, 31])])
def test_beams(dtype, K, G, page, shared):
    """Groups of beams over shared pages; each with tokens of its own."""
    lengths = [shared[s // K] + 1 + (5 * s) % 37 for s in range(2 * K)]
    check(build(dtype, lengths, 1, 2 * G, 2, 64, page, K=K, shared=shared, seed=K))


def test_dead_beams():
    """Dead slots hold no page; the first may be among them, or all of a group."""
    c = build(BF16, [50, 53, 51, 60, 61, 62, 9, 8, 7], 1, 8, 2, 128, 16, K=3, shared=[48, 32, 0])
    for s in (0, 2, 3, 4, 5):
        c["pages"][s], c["lengths"][s], c["counts"][s] = -1, 0, 0
    check(c)


def test_shared_reaches_past_the_prefix():
    """More shared tokens than some beam's prefix has are cut to it; beams with
    several asking tokens."""
    c = build(F16, [32 + 3, 32 + 5, 32 + 3, 32 + 9], 3, 4, 2, 64, 16, K=2, shared=[32, 32])
    c["shared"] = torch.tensor([1000, -4], dtype=torch.int32)
    check(c)
    c["parents"] = torch.tensor([[-1, 0, 0], [-1, -1, 1], [-1, 0, 1], [-1, 0, -1]], dtype=torch.int32)
    check(c)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_long_caches(dtype):
    """Cut over many workgroups, next to short ones."""
    check(build(dtype, [3000, 1, 0, 130], 1, 4, 2, 64, 16, seed=3))


@pytest.mark.parametrize("page", [1, 3, 7, 16, 20, 100, 1000])
def test_pages(page):
    check(build(F16, [5, 333, 64, 100], 2, 4, 2, 64, page, seed=page))


def test_many_sequences():
    """More than a wavefront has lanes, most of them idle or short."""
    lengths = [(7 * s) % 19 for s in range(150)]
    check(build(BF16, lengths, 1, 2, 1, 32, 4))


def test_pages_that_are_none():
    """Tokens whose entry is no page of the pool are seen by no query, in the
    prefix and among the asking tokens; a sequence without any page."""
    c = build(F32, [70, 70, 40, 8], 3, 4, 2, 64, 8)
    n = c["refs"].numel()
    c["pages"][0, 2], c["pages"][0, 5], c["pages"][1, 8] = -1, n, 2**31 - 1
    c["pages"][1, 0], c["pages"][2] = -2**31, n + 7
    check(c)


def test_lengths_and_counts_out_of_range():
    c = build(BF16, [40, 24, 9, 16], 4, 4, 2, 64, 8)
    c["pages"] = c["pages"][:, :5].contiguous()
    c["lengths"] = torch.tensor([41, -3, 9, 2**31 - 1], dtype=torch.int32)
    c["counts"] = torch.tensor([4, 4, -2, 2**31 - 1], dtype=torch.int32)
    c["pages"][3] = c["pages"][0]
    check(c)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N, G", [(9, 1), (40, 2), (70, 3)])
def test_values_of_unseen_branches(dtype, N, G):
    """Infinities and NaN in the keys and values of drafted tokens reach the
    rows that see them, and no other."""
    c = build(dtype, [N + 21, N], N, G, 1, 64, 16, tree=True, seed=N)
    want = expected(c)
    bad = N // 2  # of sequence 0, hidden from all that are not its descendants
    at = 21 + bad
    page, row = int(c["pages"][0, at // 16]), at % 16
    c["v"][page, row, 0, 3], c["v"][page, row, 0, 5], c["k"][page, row, 0, 0] = math.inf, math.nan, -math.inf
    out, lse = run(c)
    blind = torch.tensor([[bad not in ref.seen_by(i, N, c["parents"][s]) or s == 1 for i in range(N)] for s in range(2)])
    assert not bool(blind[0, bad]) and int(blind[0].sum()) > 0
    top = 8.0
    bound, _ = ref.attention_bounds(dtype, *want, N + 21, top)
    assert bool(((out.cpu().double() - want[0]).abs() <= bound)[blind].all())
    # a chain: the tokens ahead of it
    c["parents"] = None
    out, _ = run(c)
    out = out.cpu()
    assert bool(out[0, :bad].isfinite().all()) and bool(out[1].isfinite().all())


def test_infinite_scores():
    """Keys of -inf are left out, a row that sees only such is empty, a NaN query
    spoils its own row alone."""
    c = build(F32, [20, 20], 2, 2, 1, 32, 8)
    c["q"] = c["q"].abs() + 0.5
    for t in (0, 3, 19):
        c["k"][c["pages"][0, t // 8], t % 8, 0, 1] = -math.inf
    c["k"][c["pages"][1, :3].long()] = -math.inf
    c["q"][0, 1, 1, 4] = math.nan
    out, lse = (t.cpu() for t in run(c))
    want = expected(c)
    assert bool(out[0, 1, 1].isnan().all()) and bool(lse[0, 1, 1].isnan())
    assert bool((out[0, :, 0].double() - want[0][0, :, 0]).abs().max() < 1e-5)
    assert bool((out[1] == 0).all()) and bool(torch.isneginf(lse[1]).all())


def test_large_scores():
    """A maximum that rises all along the keys, far past the exponential's range,
    and one that is met first."""
    for sign in (1.0, -1.0):
        c = build(F32, [700], 1, 2, 1, 64, 16)
        c["q"] = torch.ones_like(c["q"])
        for t in range(700):
            c["k"][c["pages"][0, t // 16], t % 16] = sign * (t - 350) * 0.02
        check(c)


def test_layouts():
    """Keys and values of one buffer, heads ahead of tokens, queries with strides
    of their own; pools of which each page lies apart."""
    c = build(F16, [40, 90, 3], 3, 4, 2, 64, 16)
    want = expected(c)
    n = c["refs"].numel()
    joint = torch.full((n, 2, 16, 2, 64), math.nan, dtype=F16, device="cuda")
    joint[:, 0], joint[:, 1] = c["k"].cuda(), c["v"].cuda()
    check(c, run(c, k=joint[:, 0], v=joint[:, 1]), want=want)
    heads = c["k"].cuda().transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((n, 16, 2, 72), math.nan, dtype=F16, device="cuda")
    wide[..., :64] = c["v"].cuda()
    check(c, run(c, k=heads, v=wide[..., :64]), want=want)
    q = torch.empty(4, 3, 3, 64, dtype=F16, device="cuda").permute(1, 2, 0, 3)
    q.copy_(c["q"].cuda())
    check(c, run(c, q=q), want=want)
    odd = torch.empty(3 * 3 * 4 * 64 + 1, dtype=F16, device="cuda")[1:].view(3, 3, 4, 64)
    odd.copy_(c["q"].cuda())
    check(c, run(c, q=odd), want=want)
    back = c["q"].cuda().transpose(2, 3).contiguous().transpose(2, 3)
    check(c, run(c, q=back), want=want)


def test_scale_and_no_lse():
    c = build(BF16, [40, 9], 2, 4, 2, 64, 16)
    check(c, scale=0.7)
    assert torch.equal(run(c, lse=False), run(c)[0])


def test_a_pool_past_32_bits():
    """Pages more than 4 GiB into the pool."""
    page, D, n = 64, 256, 70000
    k = torch.empty(n, page, 1, D, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() * 2 > 2**31
    c = build(F16, [100, 130], 1, 2, 1, D, page)
    want = expected(c)
    small, far = c["refs"].numel(), n - 10
    k[far:far + small], v[far:far + small] = c["k"].cuda(), c["v"].cuda()
    pages = torch.where(c["pages"] >= 0, c["pages"] + far, c["pages"]).cuda()
    refs = torch.zeros(n, dtype=torch.int32, device="cuda")
    check(c, run(c, k=k, v=v, pages=pages, refs=refs), want=want)


def test_same_result_every_time_and_on_another_stream():
    c = build(BF16, [2500, 40, 700], 1, 8, 2, 128, 16)
    first = run(c)
    for _ in range(3):
        again = run(c)
        assert all(torch.equal(a, b) for a, b in zip(first, again, strict=True))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = run(c)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other, strict=True))


def test_captured():
    """A captured call follows the lengths and the cache that it reads."""
    c = build(BF16, [300, 40, 77], 1, 8, 2, 64, 16)
    cu = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    table = bg.PageTable(cu["pages"], cu["lengths"], cu["refs"])

    def call():
        return bg.tree_attention(cu["q"], cu["k"], cu["v"], table, counts=cu["counts"], return_lse=True)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for cut in (0, 37, 250, 299):
        cu["lengths"][0] = 300 - cut
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_more_sequences_than_a_launch_takes():
    """Groups of beams over several launches."""
    K = 3
    shared = [(5 * b) % 40 for b in range(110)]
    lengths = [shared[s // K] + 1 + s % 7 for s in range(110 * K)]
    check(build(BF16, lengths, 1, 2, 1, 32, 8, K=K, shared=shared))


def test_a_table_of_many_pages():
    """A table that could hold two thousand million tokens a sequence, few of them
    there: the cuts of the work stay in 31 bits."""
    c = build(F16, [2500], 1, 32, 32, 8, 1000)
    wide = torch.full((1, 2_000_000), -1, dtype=torch.int32)
    wide[:, :c["pages"].shape[1]] = c["pages"]
    want = expected(c)
    check(c, run(c, pages=wide.cuda()), want=want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_unseen_values_of_a_long_cache(dtype):
    """An infinite value in a drafted token of a sequence that several workgroups
    share."""
    N, at = 40, 1500 + 11
    c = build(dtype, [1500 + N, 30], N, 2, 1, 64, 16, tree=True, counts=[N, 0], seed=2)
    want = expected(c)
    c["v"][int(c["pages"][0, at // 16]), at % 16, 0, 7] = math.inf
    out, lse = (t.cpu().double() for t in run(c))
    bound, lse_bound = ref.attention_bounds(dtype, *want, 1500 + N, 8.0)
    for i in range(N):
        if 11 in ref.seen_by(i, N, c["parents"][0]):
            assert bool(torch.isinf(out[0, i, :, 7]).all()) and bool(out[0, i, :, :7].isfinite().all())
        else:
            assert bool(((out[0, i] - want[0][0, i]).abs() <= bound[0, i]).all())
    assert bool(((lse - want[1]).abs() <= lse_bound)[0].all())


def test_many_rows():
    """So many tiles of rows that each is one workgroup's: the ends of long prompts,
    of unlike lengths; against 64 bits on the GPU."""
    N, H, D, page = 2048, 32, 32, 32
    lengths, counts = [N + 70, N - 100], [N, 1500]
    rows = ref.sequence_rows(lengths, page)
    pages, refs = ref.make_table(rows, 1, 0)
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(2, N, H, D, device="cuda", generator=g).to(BF16)
    k, v = (torch.randn(refs.numel(), page, H, D, device="cuda", generator=g).to(BF16) for _ in range(2))
    table = bg.PageTable(pages.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), refs.cuda())
    out, lse = bg.tree_attention(q, k, v, table, counts=torch.tensor(counts).cuda(), return_lse=True)
    for s, (n, c) in enumerate(zip(lengths, counts, strict=True)):
        held = pages[s, :-(-n // page)].long().cuda()
        seen = torch.arange(n, device="cuda") <= torch.arange(c, device="cuda")[:, None] + n - c
        for h in range(0, H, 5):
            key, value = (t[held, :, h].flatten(0, 1)[:n].double() for t in (k, v))
            row = q[s, :c, h].double()
            score = (row @ key.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
            p = torch.softmax(score, -1)
            error = (row.abs() @ key.abs().T).amax(-1) / math.sqrt(D) * (D + 2) * 2.0**-24
            want = (p @ value, torch.logsumexp(score, -1), p @ value.abs(), error)
            bound, lse_bound = ref.attention_bounds(BF16, *want, n, 8.0)
            assert bool(((out[s, :c, h].double() - want[0]).abs() <= bound).all())
            assert bool(((lse[s, :c, h].double() - want[1]).abs() <= lse_bound).all())
        assert bool((out[s, c:] == 0).all()) and bool(torch.isneginf(lse[s, c:]).all())
