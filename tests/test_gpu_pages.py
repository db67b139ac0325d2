# SPDX-License-Identifier: MIT
"""The pages of a cache and the reordering of states on the GPU, against plain
restatements, value by value."""

import random

import pytest
import torch

import beamgrad_amd as bg
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make_pools(n, refs, page, shapes, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(refs.numel(), page, *shapes[i % len(shapes)], generator=g).to(dtype) for i in range(n)]


def on_gpu(pools, pages, lengths, refs):
    return [p.cuda() for p in pools], bg.PageTable(pages.cuda(), lengths.cuda(), refs.cuda())


def same(got, want):
    for a, b in zip(got, want, strict=True):
        assert torch.equal(a.cpu(), b)


def search(lengths, K, page, seed, spare):
    """Groups of K beams that share the whole pages of half their tokens."""
    rows = ref.sequence_rows(lengths, page, [min(lengths[b * K:(b + 1) * K]) // 2 for b in range(len(lengths) // K)], K)
    return ref.make_table(rows, spare, seed)


def random_parents(B, K, rng, dead=0.15):
    return torch.tensor([b * K + min(K - 1, int(rng.expovariate(3.0 / K))) if rng.random() > dead else -1
                         for b in range(B) for _ in range(K)], dtype=torch.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, K, page, spare", [(1, 1, 4, 0), (1, 4, 16, 9), (3, 5, 7, 40), (4, 8, 1, 40), (2, 16, 24, 5), (70, 16, 8, 2000)])
def test_steps(dtype, B, K, page, spare):
    """Fork, extend and write, step after step, until the pool may be full."""
    rng = random.Random(B * 100 + K)
    lengths = [rng.randrange(0, 40) for _ in range(B) for _ in range(K)]
    lengths = [lengths[s // K * K] for s in range(B * K)]  # a group's beams are as long
    pages, refs = search(lengths, K, page, B, spare)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    pools = make_pools(3, refs, page, [(2, 8), (5,)], dtype, K)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    for step in range(3):
        parents = random_parents(B, K, rng)
        pages, lengths, refs = ref.fork(pools, pages, lengths, refs, parents)
        table = bg.fork_pages(gpu, table, (parents.long() if step == 1 else parents).cuda())
        same(table, (pages, lengths, refs))
        same(gpu, pools)
        counts = torch.tensor([rng.choice([0, 1, 1, 3]) for _ in range(B * K)], dtype=torch.int32)
        before = lengths
        pages, lengths, refs = ref.extend(pages, lengths, refs, counts, page)
        table = bg.extend_pages(table, counts.cuda(), page)
        same(table, (pages, lengths, refs))
        grown = lengths - before
        news = [torch.randn(B * K, 3, *p.shape[2:], generator=torch.Generator().manual_seed(step)).to(dtype) for p in pools]
        ref.write(pools, news, pages, lengths, grown)
        bg.write_tokens(gpu, [n.cuda() for n in news], table, grown.cuda())
        same(gpu, pools)


def test_many_sequences_and_pages():
    """More sequences than the planning workgroup has threads, more pages than one
    of its rounds, few of them free."""
    rng = random.Random(5)
    S, page = 2100, 4
    lengths = torch.tensor([rng.randrange(0, 14) for _ in range(S)], dtype=torch.int32)
    pages, refs = ref.make_table(ref.sequence_rows(lengths.tolist(), page), 900, 3)
    refs[refs == 0] = (torch.arange(int((refs == 0).sum())) % 3 == 0).int()  # held by others
    pools = make_pools(1, refs, page, [(3,)], torch.float32, 1)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    parents = torch.tensor([rng.randrange(-1, S) for _ in range(S)], dtype=torch.int64)
    want = ref.fork(pools, pages, lengths, refs, parents)
    table = bg.fork_pages(gpu, table, parents.cuda())
    same(table, want)
    same(gpu, pools)
    counts = torch.tensor([rng.randrange(0, 6) for _ in range(S)], dtype=torch.int64)
    same(bg.extend_pages(table, counts.cuda(), page), ref.extend(*want, counts, page))


def test_no_page_left():
    """Forks and extensions that find no free page."""
    lengths = torch.tensor([5, 6, 7, 3], dtype=torch.int32)
    pages, refs = ref.make_table(ref.sequence_rows(lengths.tolist(), 4), 1, 0)
    pools = make_pools(2, refs, 4, [(4,)], torch.float32, 0)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    parents = torch.tensor([1, 1, 1, 3], dtype=torch.int32)
    want = ref.fork(pools, pages, lengths, refs, parents)
    got = bg.fork_pages(gpu, table, parents.cuda())
    same(got, want)
    same(gpu, pools)
    assert got.lengths.tolist() == [6, 6, 0, 3]
    for counts in ([9, 3, 0, 1], [100, 1, 4, 1], [2**31 - 1, -5, 0, 2]):
        counts = torch.tensor(counts, dtype=torch.int32)
        same(bg.extend_pages(got, counts.cuda(), 4), ref.extend(*want, counts, 4))


def test_numbers_out_of_range():
    """Parents, entries and lengths that are none: nothing is read or written for
    them."""
    lengths = torch.tensor([9, 10, 11, 6], dtype=torch.int32)
    pages, refs = ref.make_table(ref.sequence_rows(lengths.tolist(), 4), 6, 0)
    pages[2, 2], pages[0, 0], pages[3, 3] = 1000, -2**31, 2**31 - 1
    pools = make_pools(1, refs, 4, [(4,)], torch.float32, 0)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    parents = torch.tensor([2, 2, 4, 2**31 - 1], dtype=torch.int32)
    want = ref.fork(pools, pages, lengths, refs, parents)
    same(bg.fork_pages(gpu, table, parents.cuda()), want)
    same(gpu, pools)
    parents = torch.tensor([2**40, -2**40, 0, 3], dtype=torch.int64)
    want = ref.fork(pools, pages, lengths, refs, parents)
    same(bg.fork_pages(gpu, table, parents.cuda()), want)
    same(gpu, pools)
    news = [torch.randn(4, 5, 4)]
    for lengths in ([9, -1, 11, 2**31 - 1], [0, 3, 11, 20]):
        lengths = torch.tensor(lengths, dtype=torch.int32)
        ref.write(pools, news, pages, lengths, torch.tensor([5, 9, -1, 4]))
        bg.write_tokens(gpu, [n.cuda() for n in news], table._replace(lengths=lengths.cuda()),
                        torch.tensor([5, 9, -1, 4], device="cuda"))
        same(gpu, pools)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S, N, A, page, row", [(1, 1, 1, 16, 8), (3, 13, 4, 24, 20), (5, 64, 30, 7, 33), (9, 5, 9, 1, 1), (2, 40, 40, 16, 3000)])
def test_keep(dtype, S, N, A, page, row):
    rng = random.Random(N)
    lengths = [N + rng.randrange(0, 50) for _ in range(S)]
    pages, refs = ref.make_table(ref.sequence_rows(lengths, page), 2, 1)
    drafted = torch.tensor([rng.choice([N, N, max(N - 3, 0)]) for _ in range(S)], dtype=torch.int32)
    kept = torch.tensor([rng.randrange(0, min(A, max(int(d), 1)) + 1) for d in drafted], dtype=torch.int32)
    keep = torch.full((S, A), -1, dtype=torch.int32)
    for s in range(S):
        n = min(int(kept[s]), int(drafted[s]))
        keep[s, :n] = torch.tensor(sorted(rng.sample(range(int(drafted[s])), n)), dtype=torch.int32)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    pools = make_pools(3, refs, page, [(row,)], dtype, 2)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    want = ref.keep_tokens(pools, pages, lengths, refs, drafted, keep, kept)
    same(bg.keep_tokens(gpu, table, drafted.cuda(), keep.long().cuda(), kept.cuda()), want)
    same(gpu, pools)


def test_keep_of_what_is_not_drafted():
    """Lists that do not ascend or leave the draft end there; numbers out of range."""
    lengths = torch.tensor([20, 21, 22, 3, 9, 8], dtype=torch.int32)
    pages, refs = ref.make_table(ref.sequence_rows(lengths.tolist(), 4), 2, 1)
    drafted = torch.tensor([8, 8, 8, 100, -1, 8], dtype=torch.int32)
    keep = torch.tensor([[1, 3, 2, 5], [0, 8, 9, 1], [-1, 0, 1, 2], [0, 2, 3, 1], [0, 1, 2, 3], [4, 4, 5, 6]], dtype=torch.int32)
    kept = torch.tensor([4, 4, 4, 9, 4, 2**31 - 1], dtype=torch.int32)
    pools = make_pools(1, refs, 4, [(4,)], torch.float32, 2)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    want = ref.keep_tokens(pools, pages, lengths, refs, drafted, keep, kept)
    same(bg.keep_tokens(gpu, table, drafted.cuda(), keep.cuda(), kept.cuda()), want)
    same(gpu, pools)
    assert want[1].tolist() == [14, 14, 14, 2, 9, 1]


def test_layouts_and_many_pools():
    """Pools of several geometries and more than one launch holds; pages that lie
    apart, keys and values of one buffer; news with strides."""
    lengths = [9, 9, 14, 14]
    pages, refs = search(lengths, 2, 4, 0, 9)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    n = refs.numel()
    joint = torch.randn(n, 2, 4, 2, 8).cuda()
    wide = torch.randn(n, 4, 12).cuda()
    many = torch.randn(70, n, 4, 6).cuda()
    gpu = [joint[:, 0], joint[:, 1], wide[..., :5], *many.unbind(0), torch.randn(n, 4, 3).half().cuda()]
    rest = wide[..., 5:].clone()
    pools = [p.cpu().clone() for p in gpu]
    table = bg.PageTable(pages.cuda(), lengths.cuda(), refs.cuda())
    parents = torch.tensor([0, 0, 3, 3], dtype=torch.int32)
    pages, lengths, refs = ref.fork(pools, pages, lengths, refs, parents)
    table = bg.fork_pages(gpu, table, parents.cuda())
    same(table, (pages, lengths, refs))
    same(gpu, pools)
    counts = torch.tensor([3, 1, 0, 2])
    pages, lengths, refs = ref.extend(pages, lengths, refs, counts, 4)
    table = bg.extend_pages(table, counts.cuda(), 4)
    news = [torch.randn(4, 3, *p.shape[2:]).to(p.dtype) for p in pools]
    ref.write(pools, news, pages, lengths, counts)
    strided = [torch.stack([x, x], 1).cuda()[:, 0] if i % 2 else x.transpose(0, -1).contiguous().transpose(0, -1).cuda()
               for i, x in enumerate(news)]
    bg.write_tokens(gpu, strided, table, counts.cuda())
    same(gpu, pools)
    drafted, keep, kept = torch.tensor([3, 1, 0, 2]), torch.tensor([[1, 2], [0, 0], [0, 0], [1, 0]]), torch.tensor([2, 1, 0, 1])
    want = ref.keep_tokens(pools, pages, lengths, refs, drafted, keep, kept)
    same(bg.keep_tokens(gpu, table, drafted.cuda(), keep.cuda(), kept.cuda()), want)
    same(gpu, pools)
    assert torch.equal(wide[..., 5:], rest)


def test_versions_and_capture():
    """What a call writes counts as written for autograd; a captured step follows
    its inputs."""
    page, K = 4, 4
    pages, refs = search([10] * K, K, page, 0, 30)
    lengths = torch.full((K,), 10, dtype=torch.int32)
    pools = make_pools(2, refs, page, [(8,)], torch.float32, 0)
    gpu, table = on_gpu(pools, pages, lengths, refs)
    version = gpu[0]._version
    bg.fork_pages(gpu, table, torch.arange(K, dtype=torch.int32, device="cuda"))
    assert gpu[0]._version > version
    parents = torch.zeros(K, dtype=torch.int32, device="cuda")
    counts = torch.ones(K, dtype=torch.int32, device="cuda")
    news = [torch.randn(K, 1, 8, device="cuda") for _ in gpu]

    def step():
        new = bg.extend_pages(bg.fork_pages(gpu, table, parents), counts, page)
        bg.write_tokens(gpu, news, new, counts)
        return new

    start = [p.clone() for p in gpu]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for p in ([0, 0, 0, 0], [3, 1, 1, 3], [2, -1, 2, 0]):
        parents.copy_(torch.tensor(p, dtype=torch.int32))
        counts.copy_((parents >= 0).int())
        for pool, old in zip(gpu, start, strict=True):
            pool.copy_(old)
        graph.replay()
        got, wrote = [t.clone() for t in held], [p.clone() for p in gpu]
        for pool, old in zip(gpu, start, strict=True):
            pool.copy_(old)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
        assert all(torch.equal(a, b) for a, b in zip(wrote, gpu, strict=True))


# ---------------------------------------------------------------------------
# States
# ---------------------------------------------------------------------------

SHAPES = [(1, 1, ()), (1, 4, (3,)), (3, 5, (4100,)), (2, 64, (33, 5)), (2, 17, (1,)), (5, 3, (2049,)), (1, 300, (7,)), (1, 4096, (2,))]


def state_parents(B, K, seed):
    rng = random.Random(seed)
    return torch.tensor([[rng.choice([-1, k, 0, rng.randrange(K), rng.randrange(K), K + 5 if seed else 0]) for k in range(K)]
                         for _ in range(B)])


@pytest.mark.parametrize("dtype", [*DTYPES, torch.int64, torch.uint8])
@pytest.mark.parametrize("B, K, row", SHAPES)
def test_reorder(dtype, B, K, row):
    g = torch.Generator().manual_seed(K)
    states = [(torch.randn(B, K, *row, generator=g) * 50).to(dtype) for _ in range(3)] + [torch.randn(B, K, 2, generator=g)]
    parents = state_parents(B, K, K)
    want = [ref.reorder(s, parents) for s in states]
    same(bg.reorder_states([s.cuda() for s in states], parents.cuda()), want)
    gpu = [s.cuda() for s in states]
    version = gpu[0]._version
    same(bg.reorder_states(gpu, parents.int().cuda(), inplace=True), want)
    assert gpu[0]._version > version


def test_reorder_layouts():
    """Strided and expanded states, empty rows and no states; more than one launch
    holds; parts of a buffer whose neighbours stay."""
    parents = state_parents(2, 6, 1)
    base = torch.randn(2, 6, 10, 4).cuda()
    states = [base.transpose(2, 3), base[..., :3], torch.randn(2, 1, 5).cuda().expand(2, 6, 5), torch.randn(2, 6, 0).cuda()]
    same(bg.reorder_states(states, parents.cuda()), [ref.reorder(s.cpu(), parents) for s in states])
    assert bg.reorder_states([], parents.cuda()) == []
    many = torch.randn(150, 2, 6, 9).cuda()
    want = torch.stack([ref.reorder(s.cpu(), parents) for s in many])
    bg.reorder_states(list(many.unbind(0))[1:-1], parents.cuda(), inplace=True)
    assert torch.equal(many[1:-1].cpu(), want[1:-1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, K, row", SHAPES)
def test_reorder_gradient(dtype, B, K, row):
    """Against the formula: sums of up to K terms in 32 bits, rounded once."""
    g = torch.Generator().manual_seed(K)
    leaves = [torch.randn(B, K, *row, generator=g).to(dtype).cuda().requires_grad_() for _ in range(3)]
    parents = state_parents(B, K, K)
    outs = bg.reorder_states(leaves, parents.cuda())
    grads = [torch.randn(B, K, *row, generator=g).to(dtype) for _ in range(3)]
    # the last one takes no part
    got = torch.autograd.grad(outs[:2], leaves[:2], [x.cuda() for x in grads[:2]])
    for x, y in zip(got, grads, strict=False):
        want, size = ref.reorder_gradient(y, parents)
        bound = ref.HALF_STEP[dtype] * want.abs() + K * 2.0**-24 * size * 1.01 + 1e-45
        assert x.dtype == dtype and bool(((x.cpu().double() - want).abs() <= bound).all())


def test_reorder_gradient_of_differences():
    """Against differences, of a state that several beams continue, one that none
    does, a dead slot, an expanded leaf; and the gradient's own gradient."""
    parents = torch.tensor([[0, 0, -1, 1], [3, 3, 3, 3]]).cuda()
    x = torch.randn(2, 1, 5, device="cuda").requires_grad_()
    y = torch.randn(2, 4, 3, device="cuda").requires_grad_()
    w = [torch.randn(2, 4, 5, device="cuda"), torch.randn(2, 4, 3, device="cuda")]

    def loss(x, y):
        a, b = bg.reorder_states([x.expand(2, 4, 5), y], parents)
        return (a * w[0]).sum() + (b * b * w[1]).sum()

    gx, gy = torch.autograd.grad(loss(x, y), (x, y), create_graph=True)
    for t, grad in ((x, gx), (y, gy)):
        flat, step = t.detach().flatten(), 0.25
        for i in range(flat.numel()):
            ends = []
            for sign in (1, -1):
                moved = flat.clone()
                moved[i] += sign * step
                args = (moved.view_as(t), y.detach()) if t is x else (x.detach(), moved.view_as(t))
                ends.append(loss(*args).item())
            # the loss is quadratic: central differences are exact but for rounding
            assert abs((ends[0] - ends[1]) / (2 * step) - grad.flatten()[i].item()) < 1e-3
    (second,) = torch.autograd.grad(gy.sum(), y)
    want = ref.reorder_gradient((2 * w[1]).cpu(), parents.cpu())[0]
    assert torch.allclose(second.cpu().double(), want, atol=1e-5)


def test_reorder_dead_gradients_and_types():
    """What comes back for a dead slot, a NaN too, goes nowhere; states of two types."""
    parents = torch.tensor([[0, -1, 7]]).cuda()
    a = torch.randn(1, 3, 4, device="cuda").requires_grad_()
    b = torch.randn(1, 3, 4, device="cuda", dtype=torch.bfloat16).requires_grad_()
    c = torch.ones(1, 3, 2, dtype=torch.int32, device="cuda")
    outs = bg.reorder_states([a, b, c], parents)
    grads = [torch.full_like(t, float("nan")) for t in outs[:2]]
    for t in grads:
        t[:, 0] = 2.0
    got = torch.autograd.grad(outs[:2], (a, b), grads)
    for t in got:
        assert t[0, 0].tolist() == [2.0] * 4 and bool((t[0, 1:] == 0).all())


def test_reorder_captured_backward():
    """A forward and backward captured into a graph."""
    parents = torch.tensor([[0, 0, 2], [1, -1, 1]]).cuda()
    leaf = torch.randn(2, 3, 64, device="cuda").requires_grad_()
    g = torch.randn(2, 3, 64, device="cuda")

    def step():
        out = bg.reorder_states([leaf], parents)[0]
        return out.detach(), torch.autograd.grad(out, leaf, g)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = step()
    for seed in range(3):
        g.copy_(torch.randn(2, 3, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(out, want[0]) and torch.equal(grad, want[1])


def test_reorder_knows_a_leaf_of_another_stream():
    """A backward in a capture whose leaf belongs to a living graph of another
    stream would pull that stream into the capture, which ends the process: it is
    refused by this test of the leaf."""
    other = torch.ops.beamgrad.leaf_of_another_stream
    parents = torch.tensor([[0, 0, 2]]).cuda()
    leaf = torch.randn(1, 3, 64, device="cuda").requires_grad_()
    assert not other(leaf)
    alive = bg.reorder_states([leaf], parents)[0]
    assert not other(leaf)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = bg.reorder_states([leaf], parents)[0]
        assert other(leaf)
        del alive, out
        assert not other(leaf)
        out = bg.reorder_states([leaf], parents)[0]
        assert not other(leaf)
    assert other(leaf)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
