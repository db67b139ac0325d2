# SPDX-License-Identifier: MIT
"""A model's state in a search, on the GPU: a paged cache of keys and values,
the attention that reads it, and dense states in the order of the beams.

A paged cache is one pool of pages per tensor that is cached (keys and values
of every layer), ``[pages, tokens of a page, ...]``, and one
:class:`PageTable` for all of them. A step of a search:

1. :func:`fork_pages`: the new beams take over their parents' pages; only a
   last page that is not full is copied, for all but one of those that continue
   it;
2. :func:`extend_pages`: room for the new tokens;
3. :func:`write_tokens`: their keys and values;
4. :func:`tree_attention`: their attention over all that is cached, the pages
   that beams share read once.

:func:`rotary` gives queries and keys their positions ahead of 3 and 4.
:func:`accumulate_weights` sums up what attention each cached token gets, and
:func:`evict_tokens` cuts a cache to the tokens that got most of it: the prompt of
a search before its beams fork, or a long text that is scored in chunks.

:func:`keep_tokens` ends a step of speculative decoding: of a drafted tree,
whose tokens :func:`tree_attention` verified in one call, the accepted ones
stay. :func:`reorder_states` is the same for states without pages (recurrent
states, a short dense cache), with a gradient.

Every call is asynchronous on the current stream and reads nothing back: page
tables live on the GPU, so the calls can be captured into a graph. The pools (or
states in place) of a call are written at once in many places: one given twice, or
two that share memory otherwise, are refused (parts of one buffer that lie apart, in
turns too, are fine). Index tensors are int32 or int64, whose numbers
past 32 bits are out of range like any other. The C
entries are in ``include/beamgrad_state.h``. The reference has no counterpart:
its step function gathers a model's cache itself (reference
python/beamgrad/_search.py:100-133, ``BeamState.parents``).
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from types import SimpleNamespace
from typing import NamedTuple

import torch

from ._torch import _ops as _torch_ops


# the operators' only overloads: torch does not look for the one that fits
_ops = SimpleNamespace(**{name: getattr(_torch_ops, name).default for name in (
    "tree_attention", "fork_pages", "extend_pages", "write_tokens", "keep_tokens", "accumulate_weights", "evict_tokens", "rotary",
    "rotary_", "reorder_states", "reorder_states_")})


def _register_fakes() -> None:
    """Shape-only forms (torch.compile, export, meta tensors)."""

    def tree_attention(q, _k, _v, _pages, _lengths, _parents, _counts, _beams, _shared, _scale, with_lse):
        return q.new_empty(q.shape), q.new_empty(q.shape[:3] if with_lse else (0,), dtype=torch.float32)

    def table(pages, lengths, refs):
        return torch.empty_like(pages), torch.empty_like(lengths), torch.empty_like(refs)

    def fork_pages(_pools, pages, lengths, refs, _parents):
        return table(pages, lengths, refs)

    def extend_pages(pages, lengths, refs, _counts, _page_tokens):
        return table(pages, lengths, refs)

    def keep_tokens(_pools, pages, lengths, refs, *_rest):
        return table(pages, lengths, refs)

    def evict_tokens(_pools, weights, pages, lengths, refs, *_rest):
        return (*table(pages, lengths, refs), [w.new_empty(w.shape) for w in weights])

    def nothing(*_args):
        return None

    def states(tensors, *_rest):
        return [t.new_empty(t.shape) for t in tensors]

    for name, fn in (("tree_attention", tree_attention), ("fork_pages", fork_pages), ("extend_pages", extend_pages),
                     ("write_tokens", nothing), ("keep_tokens", keep_tokens), ("accumulate_weights", nothing),
                     ("evict_tokens", evict_tokens), ("rotary", states), ("rotary_", nothing), ("reorder_states", states),
                     ("reorder_states_", nothing), ("reorder_states_backward", states)):
        torch.library.register_fake(f"beamgrad::{name}", fn)


_register_fakes()


def _rotary_rule(info, in_dims, tensors, positions, frequencies, counts, *form):
    """vmap rule of rotary: the vmapped dimension becomes part of the sequences."""
    n, (of_tensors, of_positions, of_frequencies, of_counts, *_) = info.batch_size, in_dims
    if of_frequencies is not None:
        raise NotImplementedError("beamgrad_amd: vmap over the frequencies of beamgrad::rotary is not supported")

    def fold(t, dim):
        if t is None:
            return None
        return (t.unsqueeze(0).expand(n, *t.shape) if dim is None else t.movedim(dim, 0)).flatten(0, 1)

    dims = of_tensors if isinstance(of_tensors, (list, tuple)) else [of_tensors] * len(tensors)
    out = _ops.rotary([fold(t, d) for t, d in zip(tensors, dims, strict=True)], fold(positions, of_positions), frequencies,
                      fold(counts, of_counts), *form)
    return [t.unflatten(0, (n, -1)) for t in out], [0] * len(out)


torch.library.register_vmap("beamgrad::rotary", _rotary_rule)


class PageTable(NamedTuple):
    """Which pages hold the tokens of ``S`` sequences (of a search: example
    ``b``'s beam ``k`` is sequence ``b * K + k``)."""

    pages: torch.Tensor  # [S, P] int32, in order; -1 past a sequence's last page
    lengths: torch.Tensor  # [S] int32: tokens held
    refs: torch.Tensor  # [pages of the pool] int32: how many sequences hold a page; 0: it is free

    @classmethod
    def empty(cls, sequences: int, table_pages: int, pool_pages: int, device="cuda") -> PageTable:
        """The table of sequences that hold nothing yet."""
        return cls(torch.full((sequences, table_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(sequences, dtype=torch.int32, device=device),
                   torch.zeros(pool_pages, dtype=torch.int32, device=device))


def _tables(table) -> PageTable:
    if not isinstance(table, PageTable):
        raise TypeError(f"table must be a beamgrad_amd.PageTable, got {type(table).__name__}")
    return table


def _call(op, *args, **tensors):
    """``op(*args)``; where it refuses arguments that should be tensors or lists of
    them and are not, a TypeError that says which."""
    try:
        return op(*args)
    except RuntimeError:
        for name, value in tensors.items():
            many = name in ("pools", "news", "states", "tensors", "each")
            name = "weights" if name == "each" else name
            for t in value if many else (value,):
                if not isinstance(t, torch.Tensor):
                    got = type(t).__name__
                    raise TypeError(f"{name} must be a sequence of tensors, got a {got} in it" if many
                                    else f"{name} must be a torch.Tensor, got {got}") from None
        raise


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: PageTable, *,
                   parents: torch.Tensor | None = None, counts: torch.Tensor | None = None, beams: int = 1,
                   shared: torch.Tensor | None = None, scale: float | None = None, return_lse: bool = False):
    """Attention of the last tokens of each sequence over its paged cache.

    ``q`` is ``[S, N, H, D]``, the pools ``k`` and ``v`` ``[pages, tokens of a
    page, Hkv, D]`` (float32, float16 or bfloat16; ``D`` a multiple of 8 up to
    256; head ``h`` reads the cache's head ``h // (H // Hkv)``). The last
    ``counts[s]`` (default: all ``N``) of the ``table.lengths[s]`` cached tokens
    ask; their keys and values are in the cache already. Each sees the tokens
    ahead of the asking ones, itself, and

    * the asking tokens before it (a prompt's end, a single token), or
    * with ``parents`` ``[S, N]``: its ancestors in the drafted tree, node ``i``'s
      parent being node ``parents[s, i]``, -1 at a root (one that is not
      an earlier node counts as -1; at most 512 nodes).

    With ``beams`` = K > 1 the sequences come in groups of K beams whose live
    members (``counts`` > 0) hold the same pages for the whole pages of their
    first ``shared[b]`` tokens, as :func:`fork_pages` leaves them; these are
    read once for the group. ``scale`` defaults to ``1 / sqrt(D)``.

    Returns ``[S, N, H, D]`` in ``q``'s type, zeros for rows past ``counts``; with
    ``return_lse`` also the log of each row's sum of exponentials, float32
    ``[S, N, H]``, -inf for such rows. Scores, softmax and sums are held in 32
    bits; 16-bit inputs round each probability to their type. No derivatives:
    inputs that carry a tangent, or require a gradient while one is recorded, are refused.
    """
    pages, lengths, _refs = _tables(table)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    out, lse = _call(_ops.tree_attention, q, k, v, pages, lengths, parents, counts, beams, shared, scale, return_lse,
                     q=q, k=k, v=v)
    return (out, lse) if return_lse else out


def fork_pages(pools: Sequence[torch.Tensor], table: PageTable, parents: torch.Tensor) -> PageTable:
    """The table after a step of a search: sequence ``s`` continues sequence
    ``parents[s]`` (``[S]``, numbers of sequences; negative: it holds nothing).

    Whole pages are shared. A last page that is not full stays with the first
    sequence that continues its holder; each other one takes a free page and a
    copy of its tokens, in every pool (written in place). Free pages are taken in order of
    their number. A sequence that finds none is left with nothing (length 0).
    """
    pages, lengths, refs = _tables(table)
    pools = list(pools)
    return PageTable(*_call(_ops.fork_pages, pools, pages, lengths, refs, parents, pools=pools, parents=parents))


def extend_pages(table: PageTable, counts: torch.Tensor, page_tokens: int) -> PageTable:
    """Room for ``counts[s]`` (``[S]``) more tokens in pages of ``page_tokens``.

    Free pages are taken in order of their number, for the sequences in order. A
    sequence for which the pool or the table has too few keeps its pages and
    its length: ``new.lengths - table.lengths`` is what each has room for. After one
    for which the pool has too few, every later one that needs a page keeps its
    pages too. The counts of the whole pool are looked through: 0.9 us for every 1000 pages.
    """
    pages, lengths, refs = _tables(table)
    return PageTable(*_call(_ops.extend_pages, pages, lengths, refs, counts, page_tokens, counts=counts))


def write_tokens(pools: Sequence[torch.Tensor], news: Sequence[torch.Tensor], table: PageTable,
                 counts: torch.Tensor | None = None) -> None:
    """Writes ``news[i]`` (``[S, N, ...]``, a row of pool ``i`` for each token)
    to the places of the last ``counts[s]`` (default: all ``N``) tokens of each
    sequence: row ``j`` to the ``j``-th of them. These lie in pages of the sequence
    alone (:func:`extend_pages` after :func:`fork_pages` leaves them so): a page that
    several hold is written by none."""
    pages, lengths, _refs = _tables(table)
    pools, news = list(pools), list(news)
    _call(_ops.write_tokens, pools, news, pages, lengths, counts, pools=pools, news=news)


def keep_tokens(pools: Sequence[torch.Tensor], table: PageTable, drafted: torch.Tensor, keep: torch.Tensor,
                kept: torch.Tensor) -> PageTable:
    """Of the last ``drafted[s]`` tokens of each sequence, those numbered
    ``keep[s, :kept[s]]`` (``[S, A]``, ascending among the drafted ones; the
    first number that is not ends the list) stay. They move together, in place in
    every pool (so the drafted tokens lie in pages of their sequence alone, as for
    :func:`write_tokens`), and the pages that hold no token any more are given back."""
    pages, lengths, refs = _tables(table)
    pools = list(pools)
    return PageTable(*_call(_ops.keep_tokens, pools, pages, lengths, refs, drafted, keep, kept, pools=pools, drafted=drafted,
                            keep=keep, kept=kept))


def accumulate_weights(weights: torch.Tensor, q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, table: PageTable, *,
                       parents: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                       scale: float | None = None) -> None:
    """Adds up, for each cached token, the attention that the asking tokens give it.

    ``q``, ``k``, ``table``, ``parents``, ``counts`` and ``scale`` are those of a
    :func:`tree_attention`, ``lse`` (float32 ``[S, N, H]``) is what it returned with
    ``return_lse``. ``weights`` (float32 ``[S, Hkv, places]``, a place for each token that
    the table's pages can hold: ``table.pages.shape[1]`` times the tokens of a
    page) is written in place: to a token ahead of the asking ones the sum of its
    softmax weights over these and the heads that read its head is added; an asking
    token, which is new, gets its sum alone. Places past a sequence's length, and
    of tokens without a page, keep what they hold.

    Sums are held in 32 bits, in an order that does not change from run to run.
    ``reorder_states`` brings the weights ``[B, K, ...]`` of a search's beams into
    their new order. No derivatives, as :func:`tree_attention`.
    """
    pages, lengths, _refs = _tables(table)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    _call(_ops.accumulate_weights, weights, q, k, lse, pages, lengths, parents, counts, scale, weights=weights, q=q, k=k, lse=lse)


def evict_tokens(pools: Sequence[torch.Tensor], weights: Sequence[torch.Tensor], table: PageTable, budget: int | torch.Tensor, *,
                 recent: int = 0, first: int = 0) -> tuple[PageTable, list[torch.Tensor]]:
    """Cuts each sequence of more than ``budget`` tokens (an int, or ``[S]``) to
    ``budget`` of them: its last ``recent`` ones (at most ``budget``), its first ``first``
    ones (as far as the budget reaches), and of the others those with the largest
    weights, of equal ones the earlier (NaN is less than every number).

    ``weights`` (float32 ``[S, heads, places]`` each, as :func:`accumulate_weights` fills
    them) are one for each layer: as many as ``pools``, or a divisor of that, each
    then for as many pools in turn (a layer's keys and values). With ``heads`` = 1 a
    layer keeps the same tokens for all of its heads; otherwise its pools are
    ``[pages, tokens of a page, heads, ...]`` and every head keeps its own. The tokens
    that stay move together in their order, in place in every pool; the pages that hold
    none any more are given back. Returns the new table and the weights of the tokens that
    stay, zeros behind them. Positions are not lengths any more after an eviction: a
    caller of :func:`rotary` counts them by itself.

    What is written lies in pages of a sequence alone: a sequence that holds one of the
    pages to write to together with others (the prompt of a search whose beams have
    forked), or lacks a page, stays as it is; its length in the new table says so.
    """
    pages, lengths, refs = _tables(table)
    pools, weights = list(pools), list(weights)
    budgets, most = (budget, 0) if isinstance(budget, torch.Tensor) else (None, budget)
    pages, lengths, refs, weights = _call(_ops.evict_tokens, pools, weights, pages, lengths, refs, budgets, most, recent, first,
                                          pools=pools, each=weights)
    return PageTable(pages, lengths, refs), weights


def rotary_frequencies(width: int, *, base: float = 10000.0, factor: float = 1.0, context: int | None = None,
                       turns: tuple[float, float] = (1.0, 4.0), device="cuda") -> torch.Tensor:
    """The frequencies ``base ** (-2 f / width)`` of the ``width // 2`` pairs of a head,
    float64, for :func:`rotary`.

    ``factor`` stretches positions for contexts that are so many times as long as
    a model's own. Without ``context`` (tokens of the model's own) all frequencies are
    divided by it. With it, pairs that turn at least ``turns[1]`` times over the context
    keep theirs, those that turn at most ``turns[0]`` times are divided, and in
    between the two are mixed by the number of turns.
    """
    if width <= 0 or width % 2:
        raise ValueError(f"width must be a positive even number, got {width}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    half = width // 2
    own = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    stretched = own / factor
    if context is None:
        return stretched.to(device)
    low, high = turns
    if not (context > 0 and high > low):
        raise ValueError(f"context must be positive and turns ascending, got {context} and {turns}")
    keeps = ((context * own / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return torch.lerp(stretched, own, keeps).to(device)


def rotary(tensors: Sequence[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *,
           counts: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0,
           inplace: bool = False) -> list[torch.Tensor]:
    """Turns the heads of queries and keys by their tokens' positions.

    ``tensors`` are ``[S, N, H, D]`` each (``H`` and ``D`` their own; float32, float16 or
    bfloat16, of one type), ``positions`` ``[S, N]`` (int32 or int64, of any sign),
    ``frequencies`` ``[R]`` (float64; float32 is widened), as :func:`rotary_frequencies` makes them.
    The first ``2 R`` values of each head turn in pairs ``(a, b)`` by ``position *
    frequency``: values ``f`` and ``R + f``, with ``interleaved`` ``2 f`` and ``2 f + 1``. They
    are multiplied by ``scale``; the rest of a head is copied. A model that turns the end of
    its heads passes views of that. Only the first ``counts[s]`` tokens of a sequence
    count: the others become zeros.

    Sines and cosines are good to 32 bits for angles up to 2^50, of either sign. New tensors are
    returned, differentiable any number of times, in both modes. With ``inplace``
    (no derivatives) the tensors, which may be views of one buffer, are overwritten and
    returned, and the tokens past ``counts`` are not touched.
    """
    tensors = list(tensors)
    op = _ops.rotary_ if inplace else _ops.rotary
    out = _call(op, tensors, positions, frequencies, counts, interleaved, scale, False, tensors=tensors, positions=positions,
                frequencies=frequencies)
    return tensors if inplace else out


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor, *, inplace: bool = False) -> list[torch.Tensor]:
    """States ``[B, K, ...]`` in the order of the new beams: beam ``k`` of
    example ``b`` gets the row of beam ``parents[b, k]`` (``[B, K]``, as
    ``BeamState.parents``), zeros where that is negative. All states move in one
    launch.

    New tensors are returned, differentiable for float32, float16 and bfloat16:
    the gradient of a row is the sum over the beams that continue it, in their
    order and in 32 bits, rounded once; forward-mode tangents move as the states
    do. With ``inplace`` (no derivatives) the (contiguous)
    states are overwritten and returned, and rows that stay are not touched.
    """
    states = list(states)
    if inplace:
        _call(_ops.reorder_states_, states, parents, states=states, parents=parents)
        return states
    return _call(_ops.reorder_states, states, parents, states=states, parents=parents)
