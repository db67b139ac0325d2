# SPDX-License-Identifier: MIT
"""Log-probabilities of given tokens on the GPU, with entropies, alternatives and
gradients, against 64-bit restatements."""

import math

import pytest
import torch

import beamgrad_amd as bg
from tests import model_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(shape, V, dtype, seed, spread=3.0, ties=False):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(*shape, V, generator=g) * spread
    if ties:
        logits = logits.round()
    return logits.to(dtype), torch.randint(0, V, shape, generator=g)


def grads_of(shape, top, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g), torch.randn(shape, generator=g), torch.randn((*shape, top), generator=g) if top else None]


def near(got, want, bound, name=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, name
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0)), name
    far = (got - want).abs()[fine] - bound[fine]
    assert far.numel() == 0 or far.max() <= 0, (name, float(far.max()), float((got - want).abs()[fine].max()))


def check(logits, tokens, top=0, entropy=False, grads=None, place=lambda t: t.cuda()):
    """Forward, and with ``grads`` backward."""
    want, bounds = ref.token_logprobs(logits, tokens, top, entropy, grads)
    x = place(logits).detach()
    if grads is not None:
        x.requires_grad_(True)
    got = bg.token_logprobs(x, tokens.cuda(), top=top, entropy=entropy)
    near(got.logprobs, want["logprobs"], bounds["logprobs"], "logprobs")
    assert (got.entropy is None) == (not entropy) and (got.top_tokens is None) == (top == 0)
    if entropy:
        near(got.entropy, want["entropy"], bounds["entropy"], "entropy")
    if top:
        bad = torch.isnan(want["top_logprobs"])
        assert torch.equal(got.top_tokens.cpu(), torch.where(bad, -1, want["top_tokens"]))
        near(got.top_logprobs, want["top_logprobs"], bounds["top_logprobs"], "top")
    if grads is not None:
        outs = [(got.logprobs, grads[0]), (got.entropy, grads[1]), (got.top_logprobs, grads[2])]
        outs = [(o, g.cuda()) for o, g in outs if o is not None and g is not None]
        grad, = torch.autograd.grad([o for o, _ in outs], [x], [g for _, g in outs])
        assert grad.dtype == logits.dtype
        near(grad, want["grad"], bounds["grad"], "grad")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 250, 1023, 2048, 4097, 9001, 20000, 49155, 50257])
def test_rows_of_every_length(dtype, V):
    """Short rows (a wavefront), long ones, and split ones; odd lengths."""
    top = min(V, 5)
    logits, tokens = inputs((3, 2), V, dtype, V)
    check(logits, tokens, top, True, grads_of((3, 2), top, V))


@pytest.mark.parametrize("V, rows", [(40, 1100), (5000, 1030), (9001, 1), (30000, 33), (10001, 420), (50257, 60), (70001, 33)])
def test_few_and_many_rows(V, rows):
    logits, tokens = inputs((rows,), V, torch.bfloat16, rows)
    check(logits, tokens, 3, True, grads_of((rows,), 3, rows))


@pytest.mark.parametrize("V, rows", [(70001, 66), (600001, 2)])
def test_parts_of_several_rounds(V, rows):
    """Rows cut into parts that a workgroup does not read at once."""
    logits, tokens = inputs((rows,), V, torch.float32, rows)
    tokens[2::2] = -1
    check(logits, tokens, 20, True, grads_of((rows,), 20, rows))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [1, 2, 20, 63, 64])
@pytest.mark.parametrize("V", [64, 700, 12000, 49155])
def test_alternatives(dtype, top, V):
    """Ties go to the lowest token: rounded logits hold many."""
    for ties in (False, True):
        logits, tokens = inputs((4,), V, dtype, top, ties=ties)
        check(logits, tokens, top, False, [None, None, grads_of((4,), top, 3)[2]])


@pytest.mark.parametrize("V, rows", [(300, 3), (20000, 3), (50257, 3), (20000, 1100)])
def test_alternatives_of_equal_logits(V, rows):
    """More equal values than a workgroup ranks, in the whole row and beside larger ones."""
    logits = torch.zeros(rows, V)
    logits[1::3, V // 2:] = 1.0
    logits[2::3, V - 3:] = torch.tensor([2.0, 5.0, 5.0])
    logits[0, 5] = -1.0
    if rows > 3:  # (the plain form is slow)
        tokens = torch.full((rows,), -1)
        tokens[-4:] = 2
    else:
        tokens = torch.arange(rows)
    check(logits, tokens, 20, True, grads_of((rows,), 20, 1))


def test_alternatives_of_one_thread():
    """The largest values all lie where one thread of a workgroup reads."""
    for V, rows in ((2000, 2), (20000, 1030), (49155, 4)):
        logits, tokens = inputs((rows,), V, torch.float32, 1)
        tokens[:-2] = -1
        for at in range(0, V, 1024):
            logits[:, at:at + 4] += 50.0
        check(logits, tokens, 40)


def gathered(kind, rows, V, dtype, seed=0):
    """Rows whose large values lie together, or are equal in great number."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * 3
    if kind == "falling":
        x = x.sort(1, descending=True).values
    elif kind == "rising":
        x = x.sort(1).values
    elif kind == "rank":
        x = -torch.arange(1, V + 1).float().log() + 0.3 * x
    elif kind == "neighbours":
        for r, n in enumerate((600, 1000, 5000)[:rows]):
            x[r, :V // 3] = x[r, V // 3 + n:] = -math.inf
    elif kind == "turns":  # the same few threads' of every round
        x[:, torch.arange(V) % 2048 >= 60] = -math.inf
    elif kind == "negative ties":
        x = (x.clamp(max=0.0) * 2).floor() / 2 - 1.0
        x[0, ::7], x[0, 1::7] = -0.375, -0.25
        x[0, 40:] = torch.where(x[0, 40:] == -0.25, -0.375, x[0, 40:])  # fewer than are asked for stand above them
    elif kind == "wide":  # over all of the type's range, its lowest value too
        x = torch.randn(rows, V, generator=g).sign() * torch.exp(torch.rand(rows, V, generator=g) * math.log(torch.finfo(dtype).max / 4))
        x[:, ::3] = torch.finfo(dtype).min
        x[0] = torch.where(torch.arange(V) % 1000 == 3, -x[0].abs(), torch.finfo(dtype).min)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["random", "falling", "rising", "rank", "neighbours", "turns", "negative ties", "wide"])
@pytest.mark.parametrize("V", [2000, 4000, 32000, 49155, 151936])
def test_alternatives_that_lie_together(dtype, kind, V):
    """The threshold of the wavefronts' maxima lets much of the row pass: short rows (one wavefront),
    whole and split ones, of few and of all possible alternatives."""
    logits, tokens = gathered(kind, 3, V, dtype), torch.arange(3)
    for top in (5, 20, 64):
        if kind == "wide":
            # log p = (x - m) - log s rounds twice, each time to half a step of its value. The
            # restatement's bound has the first one, 2^-24 |x - m|, and multiples of log p where p is
            # not 0 in 64 bits; where it is (x - m below -745), the second, 2^-24 |log p|, comes to it
            # (its value is off by the first: 1 + 2^-23).
            want, bounds = ref.token_logprobs(logits, tokens, top, False)
            got = bg.token_logprobs(logits.cuda(), tokens.cuda(), top=top)
            assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
            for name in ("logprobs", "top_logprobs"):
                near(getattr(got, name), want[name], bounds[name] + want[name].abs() * 2.0**-24 * (1 + 2.0**-23), name)
            continue
        check(logits, tokens, top, False, [None, None, grads_of((3,), top, 1)[2]] if top == 20 and V <= 4000 else None)


def test_alternatives_of_many_rows_that_lie_together():
    """A workgroup of 256 threads a row; a split row's parts of several rounds."""
    for kind in ("falling", "rank", "turns", "negative ties"):
        logits = gathered(kind, 420, 20000, torch.bfloat16)
        tokens = torch.full((420,), -1)
        tokens[::150] = 1
        check(logits, tokens, 20)
        check(gathered(kind, 1, 1200001, torch.float32), torch.tensor([7]), 64)


@pytest.mark.parametrize("dtype, rows, V", [(torch.float32, 4, 32000), (torch.bfloat16, 32, 151936), (torch.float16, 200, 50257), (torch.float32, 600, 2000)])
def test_the_time_of_alternatives_goes_by_the_row_and_not_by_its_order(dtype, rows, V):
    """A few more passes over the row, and not two for each alternative (a hundred times as long)."""
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")

    def time(x, top):
        x, best = x.cuda(), math.inf
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(10):
                bg.token_logprobs(x, tokens, top=top)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    base = max(time(gathered("random", rows, V, dtype), 20), 0.08)  # (8 us a call: what the host takes)
    for kind in ("random", "falling", "rising", "rank", "neighbours", "turns", "negative ties"):
        took = time(gathered(kind, rows, V, dtype), 64)
        assert took <= 10 * base, (kind, took, base)


@pytest.mark.parametrize("top", [1, 6, 64])
@pytest.mark.parametrize("V, rows", [(100, 9), (20000, 9), (50257, 9), (20000, 1030)])
def test_alternatives_of_few_possible_tokens(V, rows, top):
    """Fewer of a row (and of most of its parts) are above -inf than are asked for."""
    logits, tokens = inputs((rows,), V, torch.bfloat16, 5)
    tokens[9:] = -1
    for r in range(9):
        logits[r, torch.randperm(V, generator=torch.Generator().manual_seed(r))[:V - 3 * r]] = -math.inf
    logits[8, :70], logits[7, 1:90:2] = 1.5, torch.finfo(torch.bfloat16).min
    check(logits, tokens, top, True, grads_of((rows,), top, 5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V, rows", [(100, 9), (3000, 9), (30000, 9), (49155, 9), (3000, 1030)])
def test_masked_and_invalid_rows(dtype, V, rows):
    """-inf (some, all but a few, all), the type's lowest value, NaN, +inf, tokens out of range."""
    logits, tokens = inputs((rows,), V, dtype, 4)
    tokens[9:] = -1
    logits[0, ::3] = -math.inf
    tokens[0] = 3  # masked itself
    logits[1] = -math.inf
    logits[2, 4:] = -math.inf
    logits[3] = torch.finfo(dtype).min
    logits[4, 2:] = torch.finfo(dtype).min
    logits[5, V // 2] = math.nan
    logits[6, V - 1] = math.inf
    logits[7], tokens[7] = math.nan, -1  # garbage that no token asks for
    tokens[8] = V
    check(logits, tokens, 6, True, grads_of((rows,), 6, 5))


def test_large_and_likely_tokens():
    """log p and 1 - p of a token whose probability is near 1 keep their bits."""
    logits = torch.zeros(5, 1000, dtype=torch.float32)
    logits[torch.arange(5), 7] = torch.tensor([20.0, 25.0, 30.0, 80.0, 3e38])
    tokens = torch.full((5,), 7)
    x = logits.cuda().requires_grad_(True)
    got = bg.token_logprobs(x, tokens.cuda()).logprobs
    want = torch.log_softmax(logits.double(), -1)[:, 7]
    assert ((got.cpu().double() - want).abs() <= 2.0**-22).all()
    grad, = torch.autograd.grad(got.sum(), x)
    # 1 - p = -expm1(log p), log p within 2^-22
    assert ((grad[:, 7].cpu().double() + torch.expm1(want)).abs() <= 2.0**-21).all()
    check(logits + 1000.0, tokens, 3, True, grads_of((5,), 3, 2))


def test_strides():
    """Teacher forcing's shifted rows, transposed and expanded ones, a column step."""
    logits, tokens = inputs((3, 5), 77, torch.bfloat16, 0)
    base = logits.cuda()
    cases = [(base[:, :-1], tokens[:, 1:]), (base.transpose(0, 1), tokens.T), (base[:, ::2], tokens[:, ::2]),
             (base[:1].expand(3, 5, 77), tokens), (base[:, :, 3:70], tokens.clamp(max=60)), (base[..., ::2], tokens.clamp(max=38)),
             (base[None, :, :, None].expand(2, 3, 5, 2, 77).transpose(0, 3), tokens[None, :, :, None].expand(2, 3, 5, 2)),
             (base[0, 0], tokens[0, 0])]
    for x, t in cases:
        g = grads_of(tuple(t.shape), 2, 1)
        check(x.cpu(), t, 2, True, g, place=lambda _t, x=x: x)


def test_shared_rows_sum_their_gradients():
    """An expanded leaf's gradient is the sum over its uses."""
    logits, tokens = inputs((4,), 50, torch.float32, 2)
    leaf = logits[:1].cuda().requires_grad_(True)
    bg.token_logprobs(leaf.expand(4, 50), tokens.cuda()).logprobs.sum().backward()
    p = torch.softmax(logits[0].double(), 0)
    want = torch.bincount(tokens, minlength=50).double() - 4 * p
    assert ((leaf.grad[0].cpu().double() - want).abs() <= 2.0**-20).all()


def test_index_types_and_empty_calls():
    logits, tokens = inputs((6,), 40, torch.float32, 2)
    a = bg.token_logprobs(logits.cuda(), tokens.cuda()).logprobs
    assert torch.equal(a, bg.token_logprobs(logits.cuda(), tokens.int().cuda()).logprobs)
    assert torch.equal(a[::2], bg.token_logprobs(logits[::2].cuda(), tokens.cuda()[::2]).logprobs)
    far = torch.tensor([2**32, -2**32, 2**32 + 3, -1, 40, 39]).cuda()
    got = bg.token_logprobs(logits.cuda(), far).logprobs
    assert (got[:5] == 0).all() and got[5] < 0
    none = bg.token_logprobs(torch.zeros(0, 3, 40, device="cuda", requires_grad=True), torch.zeros(0, 3, dtype=torch.int64, device="cuda"), top=2)
    assert none.logprobs.shape == (0, 3) and none.top_tokens.shape == (0, 3, 2)


def test_gradients_against_differences():
    """Central differences in the float64 restatement's logits, one direction at a time."""
    logits, tokens = inputs((2, 3), 30, torch.float32, 8, spread=1.0)
    x = logits.cuda().requires_grad_(True)
    w = grads_of((2, 3), 3, 9)

    def value(t):
        r, _ = ref.token_logprobs(t, tokens, 3, True)
        return float((r["logprobs"] * w[0]).sum() + (r["entropy"] * w[1]).sum() + (r["top_logprobs"] * w[2]).sum())

    got = bg.token_logprobs(x, tokens.cuda(), top=3, entropy=True)
    loss = (got.logprobs * w[0].cuda()).sum() + (got.entropy * w[1].cuda()).sum() + (got.top_logprobs * w[2].cuda()).sum()
    grad, = torch.autograd.grad(loss, x)
    for seed in range(5):
        d = torch.randn(2, 3, 30, generator=torch.Generator().manual_seed(seed))
        h = 2.0**-13  # the logits' own rounding to 32 bits: 2^-22 / 2^-13; the third derivative: h^2
        up, down = logits + h * d, logits - h * d
        slope = (value(up) - value(down)) / 2 / h
        assert abs(slope - float((grad.cpu().double() * d).sum())) <= 2.0**-9 * float(d.abs().sum())


def test_only_some_outputs_used():
    logits, tokens = inputs((3,), 300, torch.float32, 1)
    for use in ([0], [1], [2], [0, 2]):
        grads = [g if i in use else None for i, g in enumerate(grads_of((3,), 4, 1))]
        want, bounds = ref.token_logprobs(logits, tokens, 4, True, grads)
        x = logits.cuda().requires_grad_(True)
        got = bg.token_logprobs(x, tokens.cuda(), top=4, entropy=True)[:3]
        grad, = torch.autograd.grad([got[i] for i in use], x, [grads[i].cuda() for i in use])
        near(grad, want["grad"], bounds["grad"])


def test_derivatives_that_there_are_not():
    logits, tokens = inputs((3,), 30, torch.float32, 1)
    x = logits.cuda().requires_grad_(True)
    lp = bg.token_logprobs(x, tokens.cuda()).logprobs
    grad, = torch.autograd.grad(lp.sum(), x, create_graph=True)
    assert torch.equal(grad, torch.autograd.grad(bg.token_logprobs(x, tokens.cuda()).logprobs.sum(), x)[0])
    with pytest.raises(RuntimeError, match="no second derivative"):
        grad.sum().backward()
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda t: bg.token_logprobs(t, tokens.cuda()).logprobs, (logits.cuda(),), (logits.cuda(),))
    lp = bg.token_logprobs(x, tokens.cuda()).logprobs
    with torch.no_grad():
        x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()


def test_vmap():
    logits, tokens = inputs((4, 3), 60, torch.float32, 1)
    x, t = logits.cuda(), tokens.cuda()
    whole = bg.token_logprobs(x, t, top=3, entropy=True)

    def one(a, b):
        return tuple(bg.token_logprobs(a, b, top=3, entropy=True))

    for a, b, dims in ((x, t, (0, 0)), (x.transpose(0, 1), t, (1, 0))):
        for got, want in zip(torch.vmap(one, dims)(a, b), whole, strict=True):
            assert torch.equal(got, want)
    shared = torch.vmap(lambda b: bg.token_logprobs(x[0], b).logprobs)(t)
    assert torch.equal(shared, bg.token_logprobs(x[:1].expand(4, 3, 60), t).logprobs)
    per = torch.vmap(torch.func.grad(lambda a, b: bg.token_logprobs(a, b).logprobs.sum()))(x, t)
    leaf = x.clone().requires_grad_(True)
    bg.token_logprobs(leaf, t).logprobs.sum().backward()
    assert torch.equal(per, leaf.grad)


def test_the_same_every_time_and_on_another_stream():
    logits, tokens = inputs((64,), 20000, torch.bfloat16, 3)
    x, t = logits.cuda(), tokens.cuda()
    want = bg.token_logprobs(x, t, top=8, entropy=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = [bg.token_logprobs(x, t, top=8, entropy=True) for _ in range(4)]
    mine = [bg.token_logprobs(x, t, top=8, entropy=True) for _ in range(4)]
    torch.cuda.synchronize()
    for got in other + mine:
        for a, b in zip(got, want, strict=True):
            assert torch.equal(a, b)


def test_captured():
    """Forward and backward, replayed on new inputs; two graphs, in turns."""
    steps = []
    for rows, V in ((3, 20000), (3, 49155), (1100, 100)):
        x = torch.zeros(rows, V, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
        t = torch.zeros(rows, dtype=torch.int64, device="cuda")
        g = torch.zeros(rows, device="cuda")

        def step(x=x, t=t, g=g):
            got = bg.token_logprobs(x, t, top=4, entropy=True)
            return [*got, *torch.autograd.grad([got.logprobs, got.entropy], x, [g, g])]

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        steps.append((x, t, g, step, graph, out))
    for seed in range(3):
        for x, t, g, _step, _graph, _out in steps:
            logits, tokens = inputs(tuple(t.shape), x.shape[-1], torch.bfloat16, seed)
            with torch.no_grad():
                x.copy_(logits)
            t.copy_(tokens)
            g.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(seed)))
        for *_, graph, _out in steps:
            graph.replay()
        torch.cuda.synchronize()
        for _x, _t, _g, step, _graph, out in steps:
            for a, b in zip(out, step(), strict=True):
                assert torch.equal(a, b)


def test_a_capture_that_reaches_a_leaf_of_another_graph_is_refused():
    """The question that the capture's refusal asks, outside a capture."""
    leaf = torch.randn(2, 30, device="cuda").requires_grad_(True)
    tokens = torch.zeros(2, dtype=torch.int64, device="cuda")
    alive = bg.token_logprobs(leaf * 2, tokens).logprobs
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = bg.token_logprobs(leaf * 2, tokens).logprobs
        assert torch.ops.beamgrad.backward_reaches_leaf_of_another_stream(out)
        del alive, out
        assert not torch.ops.beamgrad.backward_reaches_leaf_of_another_stream(bg.token_logprobs(leaf, tokens).logprobs)
    torch.cuda.synchronize()


def test_a_search_rescored():
    """token_logprobs as the rescoring of beam_search, against a plain one."""
    g = torch.Generator().manual_seed(0)
    table = (torch.randn(20, 20, generator=g) * 2).cuda()
    weight = table.clone().requires_grad_(True)
    plain = table.clone().requires_grad_(True)
    options = bg.BeamOptions(beam_size=3, eos_token=4, length_penalty_alpha=0.6)

    def step(state):
        return torch.log_softmax(table[state.tokens.clamp(min=0)], -1)

    def rows(w, sequences):
        before = torch.cat([torch.zeros_like(sequences[..., :1]), sequences[..., :-1].clamp(min=0)], -1)
        return w[before]

    def own(sequences, lengths):
        return bg.token_logprobs(rows(weight, sequences), sequences).logprobs

    def other(sequences, lengths):
        lp = torch.log_softmax(rows(plain, sequences).double(), -1).gather(-1, sequences.clamp(min=0)[..., None])[..., 0]
        return torch.where(sequences >= 0, lp, 0.0)

    costs = torch.rand(2, 3, generator=g).cuda()
    grads = []
    for rescore, leaf in ((own, weight), (other, plain)):
        result = bg.beam_search(step, options, 6, batch_size=2, device="cuda", rescore_fn=rescore)
        bg.losses.minimum_risk(result, costs).backward()
        grads.append(leaf.grad)
    assert (grads[0] - grads[1]).abs().max() <= 2.0**-20
    assert grads[0].abs().max() > 0.01
