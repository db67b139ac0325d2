# SPDX-License-Identifier: MIT
"""The operators of a model's state together, as a program uses them: a beam
search with a paged cache, and a step of speculative decoding."""

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
    spec = importlib.util.spec_from_file_location("paged_beam_search", os.path.join(ROOT, "examples", "paged_beam_search.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("B, L, K, steps, page, eos", [(1, 1, 1, 5, 4, -1), (3, 21, 4, 20, 16, 5), (2, 33, 8, 30, 4, 3), (2, 16, 5, 12, 16, 2)])
def test_a_search_with_a_paged_cache(example, B, L, K, steps, page, eos):
    """The sequences of the search that runs everything again in every step."""
    model = example.Decoder(seed=K)
    prompts = torch.randint(0, 97, (B, L), device="cuda", generator=torch.Generator(device="cuda").manual_seed(L))
    options = bg.BeamOptions(beam_size=K, eos_token=eos, length_penalty_alpha=0.6)
    paged, table = example.paged_search(model, prompts, options, steps, page)
    plain = example.plain_search(model, prompts, options, steps)
    assert torch.equal(paged.sequences, plain.sequences)
    assert torch.allclose(paged.scores, plain.scores, atol=1e-4)
    # every page is counted as often as it is held
    held = torch.zeros_like(table.refs)
    pages = table.pages[table.pages >= 0].long()
    held.index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
    assert torch.equal(held, table.refs)


def test_a_step_of_speculative_decoding(example):
    """A drafted tree is verified in one call: each node's logits are those of the
    path to it alone. The accepted path stays, and decoding goes on from it."""
    model, page, S, L = example.Decoder(seed=3), 8, 2, 13
    pools = [torch.zeros(20, page, model.kv_heads, model.head, device="cuda") for _ in range(2 * model.layers)]
    table = bg.PageTable.empty(S, 6, 20)
    g = torch.Generator(device="cuda").manual_seed(0)
    prompt = torch.randint(0, 97, (S, L), device="cuda", generator=g)

    def forward(tokens, places, table, counts, parents=None):
        def attend(layer, q, k, v):
            bg.write_tokens(pools[2 * layer:2 * layer + 2], [k, v], table, counts)
            return bg.tree_attention(q, pools[2 * layer], pools[2 * layer + 1], table, parents=parents, counts=counts)
        return model.run(tokens, places, attend)

    def again(tokens):
        """The logits of one sequence, without a cache."""
        def attend(_layer, q, k, v):
            k, v = (t.repeat_interleave(2, 2).permute(0, 2, 1, 3).contiguous() for t in (k, v))
            scores = torch.matmul(q.permute(0, 2, 1, 3), k.transpose(2, 3).contiguous()) / math.sqrt(model.head)
            later = torch.ones(q.shape[1], q.shape[1], dtype=torch.bool, device="cuda").triu(1)
            return torch.matmul(torch.softmax(scores.masked_fill(later, float("-inf")), -1), v).permute(0, 2, 1, 3)
        return model.run(tokens[None], torch.arange(len(tokens), device="cuda")[None], attend)[0]

    counts = torch.full((S,), L, device="cuda")
    table = bg.extend_pages(table, counts, page)
    forward(prompt, torch.arange(L, device="cuda").expand(S, L), table, counts)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2, -1], [-1, -1, 1, 2, 3, 0, 5]], device="cuda")
    depth = torch.tensor([[0, 1, 1, 2, 2, 2, 0], [0, 0, 1, 2, 3, 1, 2]], device="cuda")
    draft = torch.randint(0, 97, (S, 7), device="cuda", generator=g)
    seven = torch.full((S,), 7, device="cuda")
    table = bg.extend_pages(table, seven, page)
    logits = forward(draft, L + depth, table, seven, parents.int())
    paths = {}
    for s in range(S):
        for i in range(7):
            path, at = [], i
            while at >= 0:
                path.insert(0, at)
                at = int(parents[s, at])
            paths[s, i] = path
            want = again(torch.cat([prompt[s], draft[s, path]]))[-1]
            assert torch.allclose(logits[s, i], want, atol=1e-4)
    # the paths to node 5 of the first and node 4 of the second sequence
    kept = [paths[0, 5], paths[1, 4]]
    keep = torch.full((S, 5), -1, device="cuda")
    for s, path in enumerate(kept):
        keep[s, :len(path)] = torch.tensor(path, device="cuda")
    many = torch.tensor([len(p) for p in kept], device="cuda")
    table = bg.keep_tokens(pools, table, seven, keep, many)
    assert table.lengths.tolist() == [L + len(p) for p in kept]
    assert int((table.refs > 0).sum()) == sum(-(-(L + len(p)) // page) for p in kept)
    one = torch.ones(S, dtype=torch.int32, device="cuda")
    last = torch.randint(0, 97, (S, 1), device="cuda", generator=g)
    before = table.lengths.long()
    table = bg.extend_pages(table, one, page)
    logits = forward(last, before[:, None], table, one)
    for s, path in enumerate(kept):
        want = again(torch.cat([prompt[s], draft[s, path], last[s]]))[-1]
        assert torch.allclose(logits[s, 0], want, atol=1e-4)


def test_compiled():
    """The operators have shapes without a GPU kernel: a traced program holds them
    as they are."""
    parents = torch.tensor([[1, 0]], device="cuda")

    @torch.compile(fullgraph=True, backend="eager")
    def step(q, k, v, pages, lengths, refs, state):
        table = bg.extend_pages(bg.PageTable(pages, lengths, refs), lengths * 0 + 1, 4)
        return bg.tree_attention(q, k, v, table, return_lse=True), bg.reorder_states([state], parents)[0]

    q, k, v = torch.randn(1, 1, 2, 32, device="cuda"), *torch.randn(2, 4, 4, 1, 32, device="cuda")
    table = bg.PageTable(*(t.cuda() for t in (torch.tensor([[2, -1]], dtype=torch.int32), torch.tensor([3], dtype=torch.int32),
                                              torch.tensor([0, 0, 1, 0], dtype=torch.int32))))
    state = torch.randn(1, 2, 5, device="cuda")
    (out, lse), moved = step(q, k, v, *table, state)
    new = bg.extend_pages(table, torch.ones(1, dtype=torch.int32, device="cuda"), 4)
    want = bg.tree_attention(q, k, v, new, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(moved, state.flip(1))
