# SPDX-License-Identifier: MIT
"""Beam search over a small decoder with a paged cache, step by step:
``python examples/paged_beam_search.py``.

The model is a stack of attention layers with random weights. Each step forks the
pages of the beams that continue several times, makes room for the new token,
writes its keys and values and attends over all that is cached, the prompt's
pages read once for all beams of an example (:func:`paged_search`). The same
search without a cache (:func:`plain_search`) runs the whole sequences through
torch again in every step; the two find the same sequences.
"""

from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import beamgrad_amd as bg  # noqa: E402


class Decoder:
    """Token embeddings, ``layers`` of attention with a residual, logits."""

    def __init__(self, vocab=97, width=64, layers=2, heads=4, kv_heads=2, head=32, longest=64, dtype=torch.float32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(*shape):
            return (torch.randn(*shape, device="cuda", generator=g) / math.sqrt(shape[-2])).to(dtype)

        self.heads, self.kv_heads, self.head, self.layers = heads, kv_heads, head, layers
        self.embed = torch.randn(vocab, width, device="cuda", generator=g).to(dtype)
        self.places = torch.randn(longest, width, device="cuda", generator=g).to(dtype)
        self.wq = [weights(width, heads * head) for _ in range(layers)]
        self.wkv = [weights(width, 2 * kv_heads * head) for _ in range(layers)]
        self.wo = [weights(heads * head, width) for _ in range(layers)]
        self.out = weights(width, vocab) * 3.0

    def run(self, tokens, places, attend):
        """Logits of ``tokens`` [S, N] at ``places`` [S, N]; ``attend(layer, q, k,
        v)`` is the attention over what came before them too."""
        S, N = tokens.shape
        x = self.embed[tokens.clamp(min=0)] + self.places[places]
        for layer in range(self.layers):
            q = (x @ self.wq[layer]).view(S, N, self.heads, self.head)
            k, v = (x @ self.wkv[layer]).view(S, N, 2, self.kv_heads, self.head).unbind(2)
            x = x + attend(layer, q, k, v).reshape(S, N, -1) @ self.wo[layer]
        return x @ self.out


def _start(prompts, options, max_steps, rows):
    """The search over ``rows(state)``, the next tokens' logits [B, K, V]."""
    def step(state):
        return torch.log_softmax(rows(state).float(), -1).view(len(prompts), options.beam_size, -1)

    with torch.no_grad():
        return bg.beam_search(step, options, max_steps, batch_size=len(prompts), device="cuda")


def paged_search(model: Decoder, prompts: torch.Tensor, options: bg.BeamOptions, max_steps: int, page: int = 16):
    """``prompts`` [B, L]; every example's beams share the pages of its prompt."""
    B, L = prompts.shape
    K = options.beam_size
    S = B * K
    width = -(-(L + max_steps) // page)
    n_pages = B * width + S * (max_steps // page + 3)
    pools = [torch.zeros(n_pages, page, model.kv_heads, model.head, dtype=model.embed.dtype, device="cuda")
             for _ in range(2 * model.layers)]
    table = bg.PageTable.empty(S, width, n_pages)
    shared = torch.full((B,), L, dtype=torch.int32, device="cuda")
    slots = torch.arange(S, device="cuda").view(B, K)

    def attend_to(table, counts, **more):
        def attend(layer, q, k, v):
            keys, values = pools[2 * layer], pools[2 * layer + 1]
            bg.write_tokens([keys, values], [k, v], table, counts)
            return bg.tree_attention(q, keys, values, table, counts=counts, **more)
        return attend

    def rows(state):
        nonlocal table
        if state.step == 0:
            # the prompt through each example's first slot, whose pages the beams
            # of the first step continue
            counts = torch.zeros(S, dtype=torch.int32, device="cuda")
            counts[slots[:, 0]] = L
            table = bg.extend_pages(table, counts, page)
            tokens = prompts.repeat_interleave(K, 0)
            logits = model.run(tokens, torch.arange(L, device="cuda").expand(S, L), attend_to(table, counts))
            return logits[:, -1]
        live = state.active.flatten()
        parents = torch.where(live, (slots[:, :1] + state.parents.clamp(min=0)).flatten(), -1)
        table = bg.fork_pages(pools, table, parents)
        before = table.lengths
        table = bg.extend_pages(table, live.int(), page)
        counts = table.lengths - before  # 0 where no page was left
        logits = model.run(state.tokens.view(S, 1), before.clamp(max=L + max_steps - 1).long().view(S, 1),
                           attend_to(table, counts, beams=K, shared=shared))
        return logits[:, -1]

    result = _start(prompts, options, max_steps, rows)
    return result, table


def plain_search(model: Decoder, prompts: torch.Tensor, options: bg.BeamOptions, max_steps: int):
    B, L = prompts.shape
    K = options.beam_size

    def attend(_layer, q, k, v):
        S, N, H, D = q.shape
        k, v = (t.repeat_interleave(H // t.shape[2], 2).float().permute(0, 2, 1, 3).contiguous() for t in (k, v))
        scores = torch.matmul(q.float().permute(0, 2, 1, 3), k.transpose(2, 3).contiguous()) / math.sqrt(D)
        later = torch.ones(N, N, dtype=torch.bool, device="cuda").triu(1)
        p = torch.softmax(scores.masked_fill(later, float("-inf")), -1)
        return torch.matmul(p, v).permute(0, 2, 1, 3).to(q.dtype)

    def rows(state):
        tokens = torch.cat([prompts.repeat_interleave(K, 0), state.sequences.reshape(B * K, -1)], 1)
        return model.run(tokens, torch.arange(tokens.shape[1], device="cuda").expand(*tokens.shape), attend)[:, -1]

    return _start(prompts, options, max_steps, rows)


def main() -> None:
    model = Decoder()
    prompts = torch.randint(0, 97, (3, 21), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    options = bg.BeamOptions(beam_size=4, eos_token=5, length_penalty_alpha=0.6)
    paged, table = paged_search(model, prompts, options, 20)
    plain = plain_search(model, prompts, options, 20)
    same = torch.equal(paged.sequences, plain.sequences)
    held = int((table.refs > 0).sum())
    print(f"best sequences {paged.sequences[:, 0, :8].tolist()} ...")
    print(f"the cache holds {held} pages of {table.refs.numel()}; the same sequences as without a cache: {same}")


if __name__ == "__main__":
    main()
