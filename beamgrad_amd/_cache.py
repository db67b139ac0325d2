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
    "tree_attention", "fork_pages", "extend_pages", "write_tokens", "keep_tokens", "reorder_states", "reorder_states_")})


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

    def nothing(*_args):
        return None

    def states(tensors, _parents):
        return [t.new_empty(t.shape) for t in tensors]

    for name, fn in (("tree_attention", tree_attention), ("fork_pages", fork_pages), ("extend_pages", extend_pages),
                     ("write_tokens", nothing), ("keep_tokens", keep_tokens), ("reorder_states", states),
                     ("reorder_states_", nothing), ("reorder_states_backward", states)):
        torch.library.register_fake(f"beamgrad::{name}", fn)


_register_fakes()


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
            many = name in ("pools", "news", "states")
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
