# SPDX-License-Identifier: MIT
"""The operators together, as a program uses them: texts read in chunks over a cache
that is cut to its heaviest tokens, and a training step that rescores them."""

import importlib.util
import math
import os

import pytest
import torch

import beamgrad_amd as bg

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("long_text", os.path.join(ROOT, "examples", "long_text.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def turn(x, positions, frequencies):
    """[N, H, D], in x's type but for the angles."""
    angle = positions.double()[:, None, None] * frequencies
    c, s = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def plain_read(model, tokens, dtype, chunk, budget, recent, first):
    """The formulas, head by head, on the CPU in `dtype`: for each text its
    log-probabilities, entropies, and of each layer and head the kept tokens with their weights."""
    w = {name: [t.detach().cpu().to(dtype) for t in getattr(model, name)] for name in ("wq", "wkv", "wo")}
    embed, last, f = model.embed.detach().cpu().to(dtype), model.out.detach().cpu().to(dtype), model.frequencies.cpu()
    H, G, D = model.heads, model.kv_heads, model.head
    texts = []
    for text in tokens.cpu():
        text = text[text >= 0]
        cache = [[{"at": torch.empty(0, dtype=torch.long), "k": torch.empty(0, D, dtype=dtype), "v": torch.empty(0, D, dtype=dtype),
                   "w": torch.empty(0, dtype=dtype)} for _ in range(G)] for _ in range(model.layers)]
        rows = []
        for begin in range(0, len(text), chunk):
            part = text[begin:begin + chunk]
            at = torch.arange(begin, begin + len(part))
            x = embed[part]
            for layer in range(model.layers):
                q = turn((x @ w["wq"][layer]).view(-1, H, D), at, f)
                k, v = (x @ w["wkv"][layer]).view(-1, 2, G, D).unbind(1)
                k = turn(k, at, f)
                outs = []
                for g in range(G):
                    c = cache[layer][g]
                    c["at"], c["k"], c["v"] = torch.cat([c["at"], at]), torch.cat([c["k"], k[:, g]]), torch.cat([c["v"], v[:, g]])
                    c["w"] = torch.cat([c["w"], torch.zeros(len(part), dtype=dtype)])
                    for h in range(g * (H // G), (g + 1) * (H // G)):
                        scores = (q[:, h] @ c["k"].T / math.sqrt(D)).masked_fill(c["at"][None] > at[:, None], -math.inf)
                        p = torch.softmax(scores, -1)
                        outs.append(p @ c["v"])
                        c["w"] = c["w"] + p.sum(0)
                x = x + torch.stack(outs, 1).reshape(len(part), -1) @ w["wo"][layer]
            rows.append(x @ last)
            for layer in cache:
                for c in layer:
                    n = len(c["at"])
                    if n <= budget:
                        continue
                    between = c["w"][first:n - recent]
                    best = torch.sort(between, descending=True, stable=True).indices[:budget - recent - first] + first
                    keep = torch.cat([torch.arange(first), best.sort().values, torch.arange(n - recent, n)])
                    for name in c:
                        c[name] = c[name][keep]
        logp = torch.log_softmax(torch.cat(rows), -1)
        texts.append((logp[:-1].gather(1, text[1:, None])[:, 0], -(logp.exp() * logp).sum(-1)[:-1], cache))
    return texts


@pytest.mark.parametrize("lengths, chunk, budget, recent, first, page, kv_heads",
                         [([61, 40, 7], 16, 24, 6, 2, 8, 2), ([90, 1], 7, 20, 0, 0, 16, 4), ([50], 50, 50, 4, 1, 16, 1), ([33, 70], 1, 9, 3, 3, 4, 2)])
def test_texts_over_a_cut_cache(example, lengths, chunk, budget, recent, first, page, kv_heads):
    """Every kept token, and scores within what 32 bits do to the plain form.

    That is taken as 32 times the plain form's own difference between 32 and 64 bits, and 32 half
    steps of the largest value: the kernels add up the same products in other orders, and
    exponentials and sines of theirs are a few half steps off where the plain form's are one."""
    model = example.Decoder(kv_heads=kv_heads, seed=len(lengths))
    tokens = torch.full((len(lengths), max(lengths)), -1)
    for s, n in enumerate(lengths):
        tokens[s, :n] = torch.randint(0, 97, (n,), generator=torch.Generator().manual_seed(s))
    logprobs, entropies, table, weights = example.read(model, tokens.cuda(), chunk=chunk, budget=budget, recent=recent, first=first, page=page)
    form = (chunk, budget, recent, first)
    exact, rough = (plain_read(model, tokens, d, *form) for d in (torch.float64, torch.float32))

    def near(got, want, other):
        if want.numel() == 0:
            return
        bound = 32 * float((want - other.double()).abs().max()) + 32 * 2.0**-24 * float(want.abs().max())
        assert float((got.cpu().double() - want).abs().max()) <= bound

    for s, n in enumerate(lengths):
        (lp, h, cache), (lp32, h32, cache32) = exact[s], rough[s]
        near(logprobs[s, :n - 1], lp, lp32)
        near(entropies[s, :n - 1], h, h32)
        assert not logprobs[s, n - 1:].any() and not entropies[s, n - 1:].any()
        assert int(table.lengths[s]) == min(n, budget)
        for layer in range(model.layers):
            for g in range(kv_heads):
                c, c32 = cache[layer][g], cache32[layer][g]
                assert torch.equal(c["at"], c32["at"])  # the choice is no matter of roundings
                near(weights[layer][s, g, :len(c["at"])], c["w"], c32["w"])
                assert not weights[layer][s, g, len(c["at"]):].any()
    held = table.pages[table.pages >= 0].long()
    assert torch.equal(table.refs, torch.zeros_like(table.refs).index_fill_(0, held, 1)) and len(held) == len(held.unique())


def test_a_cache_with_room_for_all(example):
    model = example.Decoder()
    tokens = torch.randint(0, 97, (2, 60), generator=torch.Generator().manual_seed(3)).cuda()
    tokens[1, 33:] = -1
    whole, whole_h = example.rescore(model, tokens)
    part, part_h, table, _ = example.read(model, tokens, budget=60)
    assert torch.allclose(whole, part, atol=1e-4) and torch.allclose(whole_h, part_h, atol=1e-4)
    assert table.lengths.tolist() == [60, 33]


def test_gradients_of_a_training_step(example):
    """Of every parameter, against the formulas in 64 bits, by the same measure."""
    model = example.Decoder()
    tokens = torch.randint(0, 97, (2, 21), generator=torch.Generator().manual_seed(4))
    tokens[1, 15:] = -1
    for p in model.parameters():
        p.requires_grad_(True)
    lp, h = example.rescore(model, tokens.cuda())
    grads = torch.autograd.grad(lp.sum() - 0.5 * h.sum(), model.parameters())

    def plain(dtype):
        leaves = [p.detach().cpu().to(dtype).requires_grad_(True) for p in model.parameters()]
        n = model.layers
        embed, wq, wkv, wo, out = leaves[0], leaves[1:1 + n], leaves[1 + n:1 + 2 * n], leaves[1 + 2 * n:1 + 3 * n], leaves[-1]
        H, G, D, f = model.heads, model.kv_heads, model.head, model.frequencies.cpu()
        total = 0.0
        for text in tokens:
            text = text[text >= 0]
            at = torch.arange(len(text))
            x = embed[text]
            later = at[None] > at[:, None]
            for layer in range(n):
                q = turn((x @ wq[layer]).view(-1, H, D), at, f)
                k, v = (x @ wkv[layer]).view(-1, 2, G, D).unbind(1)
                k = turn(k, at, f)
                outs = [torch.softmax((q[:, i] @ k[:, i * G // H].T / math.sqrt(D)).masked_fill(later, -math.inf), -1) @ v[:, i * G // H]
                        for i in range(H)]
                x = x + torch.stack(outs, 1).reshape(len(text), -1) @ wo[layer]
            logp = torch.log_softmax(x @ out, -1)[:-1]
            total = total + logp.gather(1, text[1:, None]).sum() + 0.5 * (logp.exp() * logp).sum()
        return torch.autograd.grad(total, leaves)

    for got, want, other in zip(grads, plain(torch.float64), plain(torch.float32), strict=True):
        bound = 32 * float((want - other.double()).abs().max()) + 32 * 2.0**-24 * float(want.abs().max())
        assert float((got.cpu().double() - want).abs().max()) <= bound


def test_the_example_runs(example, capsys):
    example.main()
    assert "pages of 8 held" in capsys.readouterr().out


def test_beams_fork_from_a_cut_prompt():
    """A prompt's cache is cut, then shared by beams; evicting it once they share it changes nothing."""
    S, heads, D, page, n = 4, 2, 16, 4, 30
    g = torch.Generator().manual_seed(0)
    keys, values = (torch.randn(40, page, heads, D, generator=g).cuda() for _ in range(2))
    pages = torch.full((S, 12), -1, dtype=torch.int32)
    pages[0, :8] = torch.arange(8)
    refs = torch.zeros(40, dtype=torch.int32)
    refs[:8] = 1
    table = bg.PageTable(pages.cuda(), torch.tensor([n, 0, 0, 0], dtype=torch.int32).cuda(), refs.cuda())
    q = torch.randn(S, 3, 4, D, generator=g).cuda()
    counts = torch.tensor([3, 0, 0, 0], dtype=torch.int32).cuda()
    weights = torch.zeros(S, heads, 12 * page, device="cuda")
    _, lse = bg.tree_attention(q, keys, values, table, counts=counts, return_lse=True)
    bg.accumulate_weights(weights, q, keys, lse, table, counts=counts)
    table, (weights,) = bg.evict_tokens([keys, values], [weights], table, 16, recent=3)
    parents = torch.zeros(S, dtype=torch.int32, device="cuda")
    table = bg.fork_pages([keys, values], table, parents)
    weights, = bg.reorder_states([weights.view(1, S, heads, -1)], parents.view(1, S))
    weights = weights.view(S, heads, -1)
    assert table.lengths.tolist() == [16] * S and torch.equal(weights[0], weights[3])
    before = [t.clone() for t in (keys, values, *table)]
    same, (after,) = bg.evict_tokens([keys, values], [weights], table, 9, recent=2)
    for got, want in zip((keys, values, *same), before, strict=True):
        assert torch.equal(got, want)
    assert torch.equal(after, weights)
    # a token more for each beam, of pages of their own
    table = bg.extend_pages(table, torch.ones(S, dtype=torch.int32, device="cuda"), page)
    new = torch.randn(2, S, 1, heads, D, generator=g).cuda()
    bg.write_tokens([keys, values], list(new), table)
    out, lse = bg.tree_attention(q[:, :1], keys, values, table, beams=S, shared=torch.full((1,), 16, dtype=torch.int32, device="cuda"), return_lse=True)
    alone, lse_alone = bg.tree_attention(q[:, :1], keys, values, table, return_lse=True)
    assert torch.allclose(out, alone, atol=1e-5) and torch.allclose(lse, lse_alone, atol=1e-5)
    total = weights.sum(-1)
    bg.accumulate_weights(weights, q[:, :1].contiguous(), keys, lse_alone, table)
    # two heads of queries for each of the cache's, a weight of one each
    assert torch.allclose(weights.sum(-1), total + 2.0, atol=1e-4)
