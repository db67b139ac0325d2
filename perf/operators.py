# SPDX-License-Identifier: MIT
"""The operators of a model's state in a beam search, as cases that a timing
program can list, draw, prepare, run and check: attention over a paged cache,
the pages of that cache, and the reordering of dense states.

A case is a dict of plain values; ``kind`` says what runs:

* ``attend``: :func:`beamgrad_amd.tree_attention`. ``B`` examples of ``K``
  beams (``K`` = 1: one sequence each), each with ``N`` tokens at the end of
  its cache that ask; ``tree``: these are a drafted tree (otherwise a chain: the
  end of a prompt); ``ragged``: sequences draft from 1 to ``N`` of them;
  ``H, Hkv, D``: heads, heads of the cache, width of a head; ``page``: tokens of a
  page; ``lo, hi``: tokens cached ahead of the asking ones (with ``K`` > 1: of
  the prompt that an example's beams share, each having ``own`` more);
  ``idle``: slots of the batch without a sequence; ``lse``: the log-sum of the
  exponentials is returned too.
* ``step``: what a step of a beam search does to the cache's pages:
  ``fork_pages``, ``extend_pages`` by one token and ``write_tokens``. ``T`` pools
  (keys and values of every layer), ``row`` values a token in each.
* ``keep``: ``keep_tokens``: of ``N`` drafted tokens a sequence, up to ``A``
  were accepted; they move together, and the pages of the others are free.
* ``reorder``: ``reorder_states`` of ``T`` states ``[B, K, row]``; ``mode``:
  ``new`` (new tensors), ``inplace``, or ``train`` (new tensors and the
  gradient).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _attend(dtype, B, K, N, H, Hkv, D, page, lo, hi, **more):
    case = dict(kind="attend", dtype=dtype, B=B, K=K, N=N, H=H, Hkv=Hkv, D=D, page=page, lo=lo, hi=hi, own=0, tree=False,
                ragged=False, idle=0, lse=False)
    case.update(more)
    return case


def _step(dtype, B, K, T, row, page, lo, hi, dead=False):
    return dict(kind="step", dtype=dtype, B=B, K=K, T=T, row=row, page=page, lo=lo, hi=hi, dead=dead)


def _keep(dtype, S, N, A, T, row, page, lo, hi):
    return dict(kind="keep", dtype=dtype, B=S, N=N, A=A, T=T, row=row, page=page, lo=lo, hi=hi)


def _reorder(dtype, B, K, T, row, mode, dead=False):
    return dict(kind="reorder", dtype=dtype, B=B, K=K, T=T, row=row, mode=mode, dead=dead)


def listed():
    cases = {
        # One user, one token, a short conversation: the latency of the call.
        "one token bf16": _attend("bfloat16", 1, 1, 1, 32, 8, 128, 16, 700, 700),
        # A step of a beam search: eight beams over each of four prompts.
        "beams bf16": _attend("bfloat16", 4, 8, 1, 32, 8, 128, 16, 2000, 6000, own=150),
        # Two readers of a book: single tokens over a very long cache.
        "long cache bf16": _attend("bfloat16", 2, 1, 1, 32, 8, 128, 64, 90000, 131000, lse=True),
        # Speculative decoding in a serving batch: ragged trees to verify.
        "drafted trees f16": _attend("float16", 8, 1, 61, 32, 8, 128, 16, 2500, 9000, tree=True, ragged=True),
        # Chunks of long prompts, narrow heads.
        "prompt chunk bf16": _attend("bfloat16", 4, 1, 1000, 32, 8, 64, 32, 1500, 4500),
        # Everything odd, in 32 bits, with an idle slot in the batch.
        "odd trees f32": _attend("float32", 5, 1, 7, 15, 5, 72, 24, 30, 1700, tree=True, idle=1, lse=True),
        # One search of four beams through a small model: latency again.
        "step few beams bf16": _step("bfloat16", 1, 4, 24, 512, 16, 90, 90),
        # A serving batch of searches through a large model's cache.
        "step many beams f16": _step("float16", 16, 8, 64, 1024, 16, 300, 900, dead=True),
        # Drafts of a few sequences, an odd page.
        "keep few f32": _keep("float32", 3, 13, 4, 12, 320, 24, 40, 400),
        # Drafts of a serving batch.
        "keep many bf16": _keep("bfloat16", 48, 64, 8, 64, 1024, 16, 200, 1200),
        # Recurrent states of a serving batch of searches, in place.
        "states in place f32": _reorder("float32", 16, 8, 24, 16384, "inplace"),
        # A training step through a search: the states' gradient too.
        "states trained bf16": _reorder("bfloat16", 8, 5, 12, 4100, "train", dead=True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """An integer of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _draw_attend(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    Hkv, G = _spread(rng, 1, 16), _spread(rng, 1, 12)
    D = 8 * _spread(rng, 4, 32)
    page = rng.choice([8, 16, 16, 20, 32, 48, 64, 128])
    form = rng.choice(["token", "token", "beams", "tree", "chunk"])
    B = _spread(rng, 1, 48 if form != "chunk" else 4)
    K, N, kept = 1, 1, 0
    if form == "beams":
        B, K, kept = _spread(rng, 1, 8), _spread(rng, 2, 16), _spread(rng, 1, 300)
    elif form == "tree":
        N = _spread(rng, 2, 100)
    elif form == "chunk":
        N = _spread(rng, 16, 1000)
    hi = _spread(rng, 1, 131000)
    # what the largest listed cases read, and what their plain forms hold
    hi = min(hi, 450_000_000 // (B * K * Hkv * max(D, 64) * _SIZE[dtype]), 19_200_000_000 // (B * K * Hkv * G * N * max(D, 64)))
    hi = max(hi, 1)
    return _attend(dtype, B, K, N, Hkv * G, Hkv, D, page, _spread(rng, 1, hi), hi, own=kept, tree=form == "tree",
                   ragged=form in ("tree", "chunk") and rng.random() < 0.5, idle=int(B > 2 and K == 1 and rng.random() < 0.4),
                   lse=rng.random() < 0.3)


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["step"] * 2 + ["keep", "reorder", "reorder"])
    if kind == "attend":
        return _draw_attend(rng)
    dtype = rng.choice(list(_TORCH))
    T = 2 * _spread(rng, 1, 32)
    row = 4 * _spread(rng, 8, 320)
    page = rng.choice([8, 16, 16, 20, 32, 64])
    if kind == "step":
        B, K = _spread(rng, 1, 32), _spread(rng, 2, 16)
        hi = _spread(rng, 1, 900)
        hi = max(1, min(hi, 250_000_000 // (B * T * row * _SIZE[dtype])))
        return _step(dtype, B, K, T, row, page, _spread(rng, 1, hi), hi, rng.random() < 0.5)
    if kind == "keep":
        N = _spread(rng, 2, 100)
        S = _spread(rng, 1, 48)
        hi = _spread(rng, 1, 1200)
        hi = max(1, min(hi, 500_000_000 // (S * T * row * _SIZE[dtype]) - N - page))
        return _keep(dtype, S, N, _spread(rng, 1, min(N, 16)), T, row, page, _spread(rng, 1, hi), hi)
    B, K, T = _spread(rng, 1, 32), _spread(rng, 2, 64), min(T, 24)
    row = max(1, min(_spread(rng, 3, 30000), 200_000_000 // (B * K * T * _SIZE[dtype])))
    return _reorder(dtype, B, K, T, row, rng.choice(["new", "inplace", "train"]), rng.random() < 0.5)


def _case_rng(case, seed=None):
    """Of a case's sizes, and with a seed of its values too."""
    sizes = [case[k] for k in sorted(case) if k != "name"]
    return random.Random(repr((sizes, seed)))


def _spaced(n, lo, hi):
    """n whole numbers of [lo, hi], evenly spread, in no order."""
    return [lo + int(math.modf((i + 0.5) * 0.6180339887498949)[0] * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    """Tokens cached ahead of the asking ones, and the asking ones, of each
    sequence of an ``attend`` case; the idle slots hold nothing."""
    B, N = case["B"], case["N"]
    ahead = _spaced(B, case["lo"], case["hi"])
    asking = _spaced(B, 1, N) if case["ragged"] else [N] * B
    for i in range(case["idle"]):
        ahead[(2 * i + 1) % B], asking[(2 * i + 1) % B] = 0, 0
    return ahead, asking


def _beam_parents(case, seed):
    """The parents of a search's step: a few beams have most children; with
    ``dead``, some examples' last slots are dead. How many children the beams
    of an example have is the case's, whose they are the seed's."""
    of_case, of_seed, K = _case_rng(case), _case_rng(case, seed), case["K"]
    rows = []
    for b in range(case["B"]):
        row = [min(K - 1, int(of_case.expovariate(3.0 / K))) for _ in range(K)]
        name = list(range(K))
        of_seed.shuffle(name)
        row = [name[p] for p in row]
        of_seed.shuffle(row)
        if case["dead"] and b % 3 == 1:
            row[-1] = -1
        rows.append(row)
    return rows


def _tree_parents(case, seed):
    """A drafted tree for each sequence: a few first guesses, each node among
    the children of a recent one."""
    rng = np.random.default_rng([seed, case["N"], case["B"]])
    B, N = case["B"], case["N"]
    at = np.arange(N)
    low = np.maximum(0, at // 2 - 2)
    parents = low + (rng.random((B, N)) * np.maximum(at - low, 1)).astype(np.int64)
    return np.where((at < 3) | (parents >= at), -1, parents).astype(np.int32)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(rows, spare, seed):
    """The page table of sequences that hold these pages (numbers from 0 up,
    shared where the same), at places of the pool in no order; and the pool's
    size, ``spare`` pages more than are held."""
    used = max((max(r) for r in rows if r), default=-1) + 1
    place = np.random.default_rng([seed, used]).permutation(used + spare).astype(np.int32)
    width = max(len(r) for r in rows) + 2
    table = np.full((len(rows), width), -1, np.int32)
    refs = np.zeros(used + spare, np.int32)
    for s, r in enumerate(rows):
        table[s, :len(r)] = place[r]
        np.add.at(refs, place[r], 1)
    return torch.from_numpy(table).cuda(), torch.from_numpy(refs).cuda(), used + spare


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_attend(case, seed):
    B, K, N, page = (case[k] for k in ("B", "K", "N", "page"))
    ahead, asking = _lengths(case)
    rows, lengths, counts, n = [], [], [], 0
    for b in range(B):
        shared = ahead[b] // page if K > 1 else 0
        first, n = list(range(n, n + shared)), n + shared
        for _ in range(K):
            length = ahead[b] + (case["own"] if asking[b] else 0) + asking[b]
            more = -(-length // page) - shared
            rows.append(first + list(range(n, n + more)))
            n += more
            lengths.append(length)
            counts.append(asking[b])
    table, refs, pages = _pages(rows, 3, seed)
    g = _generator(seed)
    dtype = _TORCH[case["dtype"]]
    pool = [torch.randn(pages, page, case["Hkv"], case["D"], device="cuda", dtype=dtype, generator=g) for _ in range(2)]
    q = torch.randn(B * K, N, case["H"], case["D"], device="cuda", dtype=dtype, generator=g) * 1.5
    return dict(q=q, k=pool[0], v=pool[1], table=(table, _int(lengths), refs),
                counts=_int(counts) if case["ragged"] or case["idle"] else None,
                parents=torch.from_numpy(_tree_parents(case, seed)).cuda() if case["tree"] else None,
                shared=_int(ahead) if K > 1 else None)


def _cache(case, seed, rows, lengths, spare):
    table, refs, pages = _pages(rows, spare, seed)
    stack = torch.randn(case["T"], pages, case["page"], case["row"], device="cuda", dtype=_TORCH[case["dtype"]],
                        generator=_generator(seed))
    return dict(stack=stack, pools=list(stack.unbind(0)), table=(table, _int(lengths), refs))


def _prepare_step(case, seed):
    B, K, page = case["B"], case["K"], case["page"]
    rows, lengths, n = [], [], 0
    for length in _spaced(B, case["lo"], case["hi"]):
        shared = length // 2 // page  # the prompt's pages
        first, n = list(range(n, n + shared)), n + shared
        for _ in range(K):
            more = -(-length // page) - shared
            rows.append(first + list(range(n, n + more)))
            n += more
            lengths.append(length)
    state = _cache(case, seed, rows, lengths, 2 * B * K)
    parents = _beam_parents(case, seed)
    state["parents"] = _int([b * K + p if p >= 0 else -1 for b, row in enumerate(parents) for p in row])
    state["counts"] = _int([int(p >= 0) for row in parents for p in row])
    state["values"] = torch.randn(case["T"], B * K, 1, case["row"], device="cuda", dtype=_TORCH[case["dtype"]],
                                  generator=_generator(seed + 1))
    state["news"] = list(state["values"].unbind(0))
    return state


def _accepted(case, seed):
    """The accepted nodes of each sequence's draft, in order: how many is the
    case's, which is the seed's."""
    S, N, A = case["B"], case["N"], case["A"]
    of_seed = _case_rng(case, seed)
    return [sorted(of_seed.sample(range(N), k)) for k in _spaced(S, 0, min(A, N))]


def _prepare_keep(case, seed):
    S, N, A, page = (case[k] for k in ("B", "N", "A", "page"))
    rows, lengths, n = [], [], 0
    for ahead in _spaced(S, case["lo"], case["hi"]):
        more = -(-(ahead + N) // page)
        rows.append(list(range(n, n + more)))
        n += more
        lengths.append(ahead + N)
    state = _cache(case, seed, rows, lengths, 3)
    keep = _accepted(case, seed)
    state["drafted"] = _int([N] * S)
    state["keep"] = _int([k + [-1] * (A - len(k)) for k in keep])
    state["kept"] = _int([len(k) for k in keep])
    return state


def _prepare_reorder(case, seed):
    T, B, K, row = (case[k] for k in ("T", "B", "K", "row"))
    dtype, g = _TORCH[case["dtype"]], _generator(seed)
    stack = torch.randn(T, B, K, row, device="cuda", dtype=dtype, generator=g)
    state = dict(stack=stack, states=list(stack.unbind(0)),
                 parents=torch.tensor(_beam_parents(case, seed), dtype=torch.int64, device="cuda"))
    if case["mode"] == "train":
        state["leaves"] = [s.clone().requires_grad_(True) for s in state["states"]]
        state["grads"] = list(torch.randn(T, B, K, row, device="cuda", dtype=dtype, generator=g).unbind(0))
    return state


_PREPARE = {"attend": _prepare_attend, "step": _prepare_step, "keep": _prepare_keep, "reorder": _prepare_reorder}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, seed), case=case)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _plain_attend(s):
    case, (pages, lengths, _refs) = s["case"], s["table"]
    S, N, H, D = s["q"].shape
    Hkv, page = case["Hkv"], case["page"]
    P = pages.shape[1]
    G, L = H // Hkv, P * page
    counts = torch.full_like(lengths, N) if s["counts"] is None else s["counts"]
    prefix = (lengths - counts).long()
    at = pages.clamp(min=0).long()
    k = s["k"][at].reshape(S, L, Hkv, D).permute(0, 2, 3, 1).float()
    q = s["q"].reshape(S, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, N * G, D).float()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).reshape(S, Hkv, N, G, L)
    del k
    # which drafted tokens each drafted token sees: itself and its ancestors
    node = torch.arange(N, device="cuda")
    if s["parents"] is None:
        sees = (node <= node[:, None]).expand(S, N, N)
    else:
        link = torch.eye(N, device="cuda") + torch.nn.functional.one_hot(s["parents"].long() + 1, N + 1)[..., 1:]
        sees = _closure(link, math.ceil(math.log2(N)))
    j = torch.arange(L, device="cuda") - prefix[:, None]  # [S, L]: the drafted token at each place, or one before or after
    drafted = (j >= 0) & (j < counts[:, None])
    visible = sees.gather(2, j.clamp(0, N - 1)[:, None, :].expand(S, N, L)) & drafted[:, None] | (j < 0)[:, None]
    visible = visible & (node < counts[:, None])[..., None]  # [S, N, L]
    scores.masked_fill_(~visible[:, None, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v"][at].reshape(S, L, Hkv, D).permute(0, 2, 1, 3).float()
    out = torch.matmul(p.reshape(S, Hkv, N * G, L), v).reshape(S, Hkv, N, G, D)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3, 4).reshape(S, N, H, D).to(s["q"].dtype)
    if not case["lse"]:
        return [out]
    return [out, (top + total.log()).squeeze(-1).permute(0, 2, 1, 3).reshape(S, N, H)]


def _closure(link, doublings):
    """Which nodes are reached over any number of links."""
    if doublings == 0:
        return link > 0
    return _closure((torch.matmul(link, link) > 0).float(), doublings - 1)


def _counted(refs, pages, by):
    """refs with ``by`` more for every page of a table."""
    return refs.clone().index_add_(0, pages.clamp(min=0).flatten().long(), by * (pages >= 0).flatten().int())


def _plain_step(s):
    pages, lengths, refs = s["table"]
    stack, page = s["stack"], s["case"]["page"]
    S, P = pages.shape
    me = torch.arange(S, device="cuda")
    # fork: full pages are shared, all but the first child copy the tail
    live = s["parents"] >= 0
    p = s["parents"].clamp(min=0).long()
    fill = lengths[p] % page
    first = torch.full((S,), S, device="cuda").scatter_reduce_(0, p, torch.where(live, me, S), "amin")
    copies = live & (fill > 0) & (first[p] != me)
    free = torch.argsort((refs > 0).int(), stable=True)  # the free pages, in order
    n_free = (refs == 0).sum()
    rank = copies.long().cumsum(0) - 1
    live = live & ~(copies & (rank >= n_free))
    copies = copies & live
    fresh = free[rank.clamp(0, free.numel() - 1)].int()
    tail = (lengths[p] // page).clamp(max=P - 1).long()
    forked = torch.where(live[:, None], pages[p], -1)
    to = torch.where(copies[:, None] & (torch.arange(P, device="cuda") == tail[:, None]), fresh[:, None], forked)
    child, offset = (copies[:, None] & (torch.arange(page, device="cuda") < fill[:, None])).nonzero(as_tuple=True)
    source = forked[child, tail[child]].long()
    stack[:, fresh[child].long(), offset] = stack[:, source, offset]
    pages = to
    refs = _counted(_counted(refs, s["table"][0], -1), pages, 1)
    lengths = torch.where(live, lengths[p], 0)
    # extend by a token
    counts = s["counts"]
    column = torch.arange(P, device="cuda")
    held, wanted = -(-lengths // page), -(-(lengths + counts) // page)
    fits = wanted <= P
    fresh_at = (column >= held[:, None]) & (column < wanted[:, None]) & fits[:, None]
    free = torch.argsort((refs > 0).int(), stable=True)
    n_free = (refs == 0).sum()
    rank = fresh_at.flatten().long().cumsum(0).reshape(S, P) - 1
    fits = fits & ~(fresh_at & (rank >= n_free)).any(1)
    fresh_at = fresh_at & fits[:, None]
    pages = torch.where(fresh_at, free[rank.clamp(0, free.numel() - 1)].int(), pages)
    refs = _counted(refs, torch.where(fresh_at, pages, -1), 1)
    lengths = torch.where(fits, lengths + counts, lengths)
    # write the new tokens
    who = (fits & (counts > 0)).nonzero().squeeze(1)
    last = (lengths[who] - 1).long()
    stack[:, pages[who, last // page].long(), last % page] = s["values"][:, who, 0]
    return [stack, pages, lengths, refs]


def _plain_keep(s):
    pages, lengths, refs = s["table"]
    stack, page = s["stack"], s["case"]["page"]
    start = lengths - s["drafted"]
    A = s["keep"].shape[1]
    i = torch.arange(A, device="cuda")
    who, i = (i < s["kept"][:, None]).nonzero(as_tuple=True)
    source = (start[who] + s["keep"][who, i]).long()
    to = start[who].long() + i
    stack[:, pages[who, to // page].long(), to % page] = stack[:, pages[who, source // page].long(), source % page]
    lengths = start + s["kept"]
    kept = torch.where(torch.arange(pages.shape[1], device="cuda") < -(-lengths // page)[:, None], pages, -1)
    return [stack, kept, lengths, _counted(_counted(refs, pages, -1), kept, 1)]


def _plain_reorder(s):
    case, parents = s["case"], s["parents"]
    b = torch.arange(case["B"], device="cuda")[:, None]
    p = parents.clamp(min=0)
    dead = (parents < 0)[..., None]
    if case["mode"] == "inplace":
        s["stack"].copy_(s["stack"][:, b, p].masked_fill(dead, 0.0))
        return [s["stack"]]
    news = [x[b, p].masked_fill(dead, 0.0) for x in s["states"]]
    if case["mode"] == "new":
        return news
    flat = (p + b * case["K"]).flatten()
    zeros = torch.zeros(case["B"] * case["K"], case["row"], device="cuda")
    gradients = [zeros.index_add(0, flat, g.float().masked_fill(dead, 0.0).flatten(0, 1)).to(g.dtype) for g in s["grads"]]
    return news + [g.unflatten(0, (case["B"], case["K"])) for g in gradients]


_PLAIN = {"attend": _plain_attend, "step": _plain_step, "keep": _plain_keep, "reorder": _plain_reorder}


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------


def _own_attend(s):
    import beamgrad_amd as bg

    return bg.tree_attention(s["q"], s["k"], s["v"], bg.PageTable(*s["table"]), parents=s["parents"], counts=s["counts"],
                             beams=s["case"]["K"], shared=s["shared"], return_lse=s["case"]["lse"])


def _own_step(s):
    import beamgrad_amd as bg

    table = bg.fork_pages(s["pools"], bg.PageTable(*s["table"]), s["parents"])
    table = bg.extend_pages(table, s["counts"], s["case"]["page"])
    bg.write_tokens(s["pools"], s["news"], table, s["counts"])
    return [s["stack"], *table]


def _own_keep(s):
    import beamgrad_amd as bg

    return [s["stack"], *bg.keep_tokens(s["pools"], bg.PageTable(*s["table"]), s["drafted"], s["keep"], s["kept"])]


def _own_reorder(s):
    import beamgrad_amd as bg

    mode = s["case"]["mode"]
    if mode == "inplace":
        bg.reorder_states(s["states"], s["parents"], inplace=True)
        return [s["stack"]]
    if mode == "new":
        return bg.reorder_states(s["states"], s["parents"])
    news = bg.reorder_states(s["leaves"], s["parents"])
    return [*news, *torch.autograd.grad(news, s["leaves"], s["grads"])]


_OWN = {"attend": _own_attend, "step": _own_step, "keep": _own_keep, "reorder": _own_reorder}


def run(state):
    out = (_OWN if own else _PLAIN)[state["case"]["kind"]](state)
    return list(out) if isinstance(out, (list, tuple)) else [out]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _work_attend(case):
    ahead, asking = _lengths(case)
    B, K, H, D = (case[k] for k in ("B", "K", "H", "D"))
    parents = _tree_parents(case, 0) if case["tree"] else None
    tokens = pairs = 0
    for b in range(B):
        n, mine = asking[b], case["own"] if asking[b] else 0
        tokens += ahead[b] + K * (mine + n)
        if parents is None:
            seen = n * (n + 1) // 2
        else:
            depth = []
            for i in range(n):
                depth.append(1 + (depth[parents[b, i]] if parents[b, i] >= 0 else 0))
            seen = sum(depth)
        pairs += K * (n * (ahead[b] + mine) + seen)
    queries = B * K * case["N"] * H * D
    out = 2 * queries * _SIZE[case["dtype"]] + (4 * queries // D if case["lse"] else 0)
    return {"bytes": 2 * tokens * case["Hkv"] * D * _SIZE[case["dtype"]] + out, "flops": 4 * D * H * pairs}


def work(case):
    if case["kind"] == "attend":
        return _work_attend(case)
    size = _SIZE[case["dtype"]]
    if case["kind"] == "reorder":
        parents = _beam_parents(case, 0)
        rows = case["T"] * case["row"] * size
        read = sum(len({p for p in row if p >= 0}) for row in parents)
        written = sum(map(len, parents))
        if case["mode"] == "inplace":  # rows that stay where they are need no work
            moved = [(k, p) for row in parents for k, p in enumerate(row) if p != k]
            read = sum(len({p for k, p in enumerate(row) if p >= 0 and p != k}) for row in parents)
            written = len(moved)
        train = 2 if case["mode"] == "train" else 1
        adds = sum(p >= 0 for row in parents for p in row) * case["T"] * case["row"] if train == 2 else 0
        return {"bytes": train * (read + written) * rows, "flops": adds}
    table = 4 * case["B"] * case.get("K", 1) * (-(-(case["hi"] + case.get("N", 1)) // case["page"]) + 2)
    token = case["T"] * case["row"] * size
    if case["kind"] == "keep":
        moved = sum(int(k != i) for keep in _accepted(case, 0) for i, k in enumerate(keep))
        return {"bytes": 2 * moved * token + 4 * table, "flops": 0}
    moved = 0
    for length, row in zip(_spaced(case["B"], case["lo"], case["hi"]), _beam_parents(case, 0), strict=True):
        live = [p for p in row if p >= 0]
        moved += (len(live) - len(set(live))) * (length % case["page"]) + len(live)
    return {"bytes": 2 * moved * token + 4 * table, "flops": 0}


# ---------------------------------------------------------------------------
# The results by the definitions, one sequence, row or token after the other
# ---------------------------------------------------------------------------


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    S, N, H, D = s["q"].shape
    G, page = H // case["Hkv"], case["page"]
    pages, lengths = s["table"][0].tolist(), s["table"][1].tolist()
    counts = s["counts"].tolist() if s["counts"] is not None else [N] * S
    parents = s["parents"].tolist() if s["parents"] is not None else None
    out = torch.zeros(S, N, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((S, N, H), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(S):
        n, c = lengths[b], counts[b]
        if c == 0:
            continue
        held = torch.tensor(pages[b][:-(-n // page)], device="cuda")
        keys = s["k"][held].flatten(0, 1)[:n]
        values = s["v"][held].flatten(0, 1)[:n]
        hidden = np.zeros((c, n), bool)
        for i in range(c):
            line, at = set(), i
            while parents is not None and at >= 0:
                line.add(at)
                at = parents[b][at]
            hidden[i, n - c:] = [(j not in line) if parents is not None else (j > i) for j in range(c)]
        hidden = torch.from_numpy(hidden).cuda()
        for h in range(H):
            key, value = keys[:, h // G].double(), values[:, h // G].double()
            score = (s["q"][b, :c, h].double() @ key.T) / math.sqrt(D)
            score[hidden] = -math.inf
            lse[b, :c, h] = torch.logsumexp(score, -1)
            out[b, :c, h] = torch.softmax(score, -1) @ value
    return [out, lse] if case["lse"] else [out]


def _exact_step(case, seed):
    s = _prepare_step(case, seed)
    pages, lengths, refs = (t.tolist() for t in s["table"])
    page, stack, count = case["page"], s["stack"], list(refs)
    free = [i for i, r in enumerate(refs) if r == 0]
    taken, moves, kids = 0, [], set()
    new_pages, new_lengths = [], []
    for row in pages:
        for at in row:
            if at >= 0:
                count[at] -= 1
    for child, parent in enumerate(s["parents"].tolist()):
        row, n = ([-1] * len(pages[0]), 0) if parent < 0 else (list(pages[parent]), lengths[parent])
        if n % page and parent in kids:
            moves.append((row[n // page], free[taken], n % page))
            row[n // page] = free[taken]
            taken += 1
        kids.add(parent)
        new_pages.append(row)
        new_lengths.append(n)
    for row in new_pages:
        for at in row:
            if at >= 0:
                count[at] += 1
    source = torch.tensor([[a, i] for a, _, n in moves for i in range(n)], dtype=torch.long, device="cuda").reshape(-1, 2)
    to = torch.tensor([[b, i] for _, b, n in moves for i in range(n)], dtype=torch.long, device="cuda").reshape(-1, 2)
    stack[:, to[:, 0], to[:, 1]] = stack[:, source[:, 0], source[:, 1]]
    free = iter([i for i, r in enumerate(count) if r == 0])
    puts = []
    for child, more in enumerate(s["counts"].tolist()):
        if not more:
            continue
        n = new_lengths[child]
        if n % page == 0:
            new_pages[child][n // page] = next(free)
            count[new_pages[child][n // page]] += 1
        puts.append((child, new_pages[child][n // page], n % page))
        new_lengths[child] = n + 1
    put = torch.tensor(puts, dtype=torch.long, device="cuda").reshape(-1, 3)
    stack[:, put[:, 1], put[:, 2]] = s["values"][:, put[:, 0], 0]
    return [stack, _int(new_pages), _int(new_lengths), _int(count)]


def _exact_keep(case, seed):
    s = _prepare_keep(case, seed)
    pages, lengths, count = (t.tolist() for t in s["table"])
    page, stack, moves = case["page"], s["stack"], []
    for b, keep in enumerate(_accepted(case, seed)):
        start = lengths[b] - case["N"]
        for i, node in enumerate(keep):
            a, z = start + node, start + i
            moves.append((pages[b][a // page], a % page, pages[b][z // page], z % page))
        lengths[b] = start + len(keep)
        for j in range(-(-lengths[b] // page), len(pages[b])):
            if pages[b][j] >= 0:
                count[pages[b][j]] -= 1
                pages[b][j] = -1
    m = torch.tensor(moves, dtype=torch.long, device="cuda").reshape(-1, 4)
    stack[:, m[:, 2], m[:, 3]] = stack[:, m[:, 0], m[:, 1]]
    return [stack, _int(pages), _int(lengths), _int(count)]


def _exact_reorder(case, seed):
    s = _prepare_reorder(case, seed)
    parents = _beam_parents(case, seed)
    news = torch.zeros(case["T"], case["B"], case["K"], case["row"], dtype=torch.float64, device="cuda")
    back = torch.zeros_like(news)
    for b, row in enumerate(parents):
        for k, p in enumerate(row):
            if p >= 0:
                news[:, b, k] = s["stack"][:, b, p].double()
                if case["mode"] == "train":
                    back[:, b, p] += torch.stack([g[b, k] for g in s["grads"]]).double()
    if case["mode"] == "inplace":
        return [news]
    return [*news.unbind(0), *(back.unbind(0) if case["mode"] == "train" else ())]


def exact(case, seed):
    return {"attend": _exact_attend, "step": _exact_step, "keep": _exact_keep, "reorder": _exact_reorder}[case["kind"]](case, seed)
