# SPDX-License-Identifier: MIT
"""Long texts in a small cache: ``python examples/long_text.py``.

The model is a stack of attention layers with random weights and rotary positions.
:func:`read` goes through texts in chunks. After each one, the cache is cut to the
tokens that got most of the attention so far, each head's its own, beside the first
and the last ones: what it holds, and what a token costs, does not grow with the
text. It returns every token's log-probability and the entropy of what was expected
there. :func:`rescore` is the same without a cache and with gradients, as a training
step has it; where the cache has room for the whole text the two agree.
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

    def __init__(self, vocab=97, width=64, layers=2, heads=4, kv_heads=2, head=32, dtype=torch.float32, seed=0):
        g = torch.Generator().manual_seed(seed)

        def weights(*shape):
            return (torch.randn(*shape, generator=g) / math.sqrt(shape[-2])).to("cuda", dtype)

        self.heads, self.kv_heads, self.head, self.layers = heads, kv_heads, head, layers
        self.frequencies = bg.rotary_frequencies(head)
        self.embed = weights(vocab, width) * math.sqrt(vocab)
        self.wq = [weights(width, heads * head) * 2.0 for _ in range(layers)]
        self.wkv = [weights(width, 2 * kv_heads * head) for _ in range(layers)]
        self.wo = [weights(heads * head, width) for _ in range(layers)]
        self.out = weights(width, vocab) * 2.0

    def parameters(self):
        return [self.embed, *self.wq, *self.wkv, *self.wo, self.out]

    def run(self, tokens, positions, attend, counts=None):
        """Logits of ``tokens`` [S, N] (negative ones count as 0) at ``positions``; ``attend(layer,
        q, k, v)`` is the attention over what came before them too."""
        S, N = tokens.shape
        x = self.embed[tokens.clamp(min=0)]
        for layer in range(self.layers):
            q = (x @ self.wq[layer]).view(S, N, self.heads, self.head)
            k, v = (x @ self.wkv[layer]).view(S, N, 2, self.kv_heads, self.head).unbind(2)
            q, k = bg.rotary([q, k], positions, self.frequencies, counts=counts)
            x = x + attend(layer, q, k, v).reshape(S, N, -1) @ self.wo[layer]
        return x @ self.out


def read(model: Decoder, tokens: torch.Tensor, *, chunk: int = 16, budget: int = 32, recent: int = 8, first: int = 2, page: int = 8):
    """``tokens`` [S, L], -1 past a text's end, in chunks over a cache of ``budget``
    tokens. Returns the log-probability of each token after the first of its text
    [S, L - 1] and the entropies there, the page table and the attention weights
    of what is cached."""
    S, L = tokens.shape
    width = -(-(budget + chunk) // page)
    n_pages = S * (width + 1)
    dtype, device = model.embed.dtype, tokens.device
    pools = [torch.zeros(n_pages, page, model.kv_heads, model.head, dtype=dtype, device=device) for _ in range(2 * model.layers)]
    weights = [torch.zeros(S, model.kv_heads, width * page, device=device) for _ in range(model.layers)]
    table = bg.PageTable.empty(S, width, n_pages)
    lengths = (tokens >= 0).sum(1)
    logprobs, entropies = [], []
    with torch.no_grad():
        for begin in range(0, L, chunk):
            part = tokens[:, begin:begin + chunk]
            counts = (lengths - begin).clamp(0, part.shape[1])
            table = bg.extend_pages(table, counts, page)

            def attend(layer, q, k, v, table=table, counts=counts):
                keys, values = pools[2 * layer], pools[2 * layer + 1]
                bg.write_tokens([keys, values], [k, v], table, counts)
                out, lse = bg.tree_attention(q, keys, values, table, counts=counts, return_lse=True)
                bg.accumulate_weights(weights[layer], q, keys, lse, table, counts=counts)
                return out

            positions = torch.arange(begin, begin + part.shape[1], device=device).expand(part.shape)
            logits = model.run(part, positions, attend, counts)
            follows = torch.full_like(part, -1)
            after = tokens[:, begin + 1:begin + 1 + part.shape[1]]
            follows[:, :after.shape[1]] = after
            scores = bg.token_logprobs(logits, follows, entropy=True)
            logprobs.append(scores.logprobs)
            entropies.append(scores.entropy)
            table, weights = bg.evict_tokens(pools, weights, table, budget, recent=recent, first=first)
    return torch.cat(logprobs, 1)[:, :-1], torch.cat(entropies, 1)[:, :-1], table, weights


def rescore(model: Decoder, tokens: torch.Tensor):
    """Log-probabilities and entropies as :func:`read` returns, of all tokens at
    once, and differentiable."""
    S, N = tokens.shape
    later = torch.ones(N, N, dtype=torch.bool, device=tokens.device).triu(1)

    def attend(_layer, q, k, v):
        k, v = (t.repeat_interleave(model.heads // model.kv_heads, 2).float().transpose(1, 2) for t in (k, v))
        scores = torch.matmul(q.float().transpose(1, 2), k.transpose(2, 3).contiguous()) / math.sqrt(model.head)
        return torch.matmul(torch.softmax(scores.masked_fill(later, -math.inf), -1), v.contiguous()).transpose(1, 2).to(q.dtype)

    logits = model.run(tokens, torch.arange(N, device=tokens.device).expand(S, N), attend)
    scores = bg.token_logprobs(logits[:, :-1], tokens[:, 1:], entropy=True)
    return scores.logprobs, scores.entropy


def main() -> None:
    model = Decoder()
    tokens = torch.randint(0, 97, (3, 200), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    tokens[1, 120:] = -1
    for p in model.parameters():
        p.requires_grad_(True)
    whole, _ = rescore(model, tokens)
    loss = -whole.sum() / (tokens[:, 1:] >= 0).sum()
    grads = torch.autograd.grad(loss, model.parameters())
    print(f"loss of all tokens at once: {float(loss.detach()):.4f}, of a gradient of norm {float(sum((g ** 2).sum() for g in grads)) ** 0.5:.4f}")
    for budget in (200, 64, 32):
        part, _, table, _ = read(model, tokens, budget=budget)
        print(f"a cache of {budget} tokens: loss {float(-part.sum() / (tokens[:, 1:] >= 0).sum()):.4f}, "
              f"{int((table.refs > 0).sum())} pages of 8 held at the end")


if __name__ == "__main__":
    main()
