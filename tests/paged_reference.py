# SPDX-License-Identifier: MIT
"""Plain restatements of the operators of a model's state (attention over a
paged cache, the cache's pages, reordering of states), on the CPU: attention
in 64 bits, one row after the other; pages and rows moved one by one."""

from __future__ import annotations

import math
import random

import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def make_table(rows, spare, seed, extra=2):
    """A page table of sequences that hold these pages (numbers from 0, shared
    where equal), at shuffled places of a pool with ``spare`` pages more."""
    used = max((max(r) for r in rows if r), default=-1) + 1
    place = list(range(used + spare))
    random.Random(seed).shuffle(place)
    width = max(1, max(len(r) for r in rows) + extra)
    pages = torch.full((len(rows), width), -1, dtype=torch.int32)
    refs = torch.zeros(used + spare, dtype=torch.int32)
    for s, r in enumerate(rows):
        for c, page in enumerate(r):
            pages[s, c] = place[page]
            refs[place[page]] += 1
    return pages, refs


def sequence_rows(lengths, page, shared=None, K=1):
    """Pages of each sequence; with ``shared`` (tokens, one entry a group of K) the
    group's first whole pages are the same."""
    rows, n = [], 0
    for s, length in enumerate(lengths):
        if K > 1 and s % K == 0:
            whole = shared[s // K] // page if shared is not None else 0
            common, n = list(range(n, n + whole)), n + whole
        held = -(-length // page)
        mine = common[:held] if K > 1 else []
        more = held - len(mine)
        rows.append(mine + list(range(n, n + more)))
        n += more
    return rows


def seen_by(i, count, parents):
    """The asking tokens that asking token i sees."""
    if parents is None:
        return list(range(i + 1))
    line, at = [], i
    while at >= 0:
        line.append(at)
        up = int(parents[at])
        at = up if 0 <= up < at else -1
    return line


def attention(q, k, v, pages, lengths, counts, parents, scale):
    """(out, lse, magnitude, score error) in float64: magnitude is sum p |v|, the
    score error a bound of the float32 products' and sums' on any score of a row."""
    S, N, H, D = q.shape
    n_pages, page, Hkv, _ = k.shape
    out = torch.zeros(S, N, H, D, dtype=torch.float64)
    magnitude = torch.zeros_like(out)
    lse = torch.full((S, N, H), -math.inf, dtype=torch.float64)
    error = torch.zeros(S, N, H, dtype=torch.float64)
    for s in range(S):
        length = min(max(int(lengths[s]), 0), pages.shape[1] * page)
        count = min(max(int(counts[s]), 0), N, length)
        at = []
        for t in range(length):
            entry = int(pages[s, t // page])
            at.append((entry, t % page) if 0 <= entry < n_pages else None)
        for i in range(count):
            tokens = list(range(length - count)) + [length - count + j for j in sorted(seen_by(i, count, None if parents is None else parents[s]))]
            places = [at[t] for t in tokens if at[t] is not None]
            if not places:
                continue
            a, b = (torch.tensor(x) for x in zip(*places, strict=True))
            for h in range(H):
                key, value = k[a, b, h // (H // Hkv)].double(), v[a, b, h // (H // Hkv)].double()
                row = q[s, i, h].double()
                score = key @ row * scale
                lse[s, i, h] = torch.logsumexp(score, 0)
                p = torch.softmax(score, 0)
                out[s, i, h] = p @ value
                magnitude[s, i, h] = p @ value.abs()
                error[s, i, h] = (key.abs() @ row.abs()).max() * scale * (D + 2) * 2.0**-24
    return out, lse, magnitude, error


def attention_bounds(dtype, out, lse, magnitude, error, longest, top_value):
    """How far a kernel may be from `attention`: the scores' error moves each
    probability by a factor of e^(2 error) at most (itself and the total); the
    exponential and the sums of up to `longest` terms in float32 (and their rescaling)
    round by 2^-24 a step, the exponential by some of them; a 16-bit type
    rounds each probability, and its least step bounds small ones (the largest of a
    row is 1 or more); the result is rounded once."""
    half = HALF_STEP[dtype]
    steps = (2 * longest + 64) * 2.0**-24
    p_error = half if dtype != torch.float32 else 0.0
    grow = torch.expm1(2 * error)[..., None]
    least = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}[dtype]
    bound = half * out.abs() + (p_error + grow + steps) * magnitude * (1 + half) + least * (1 + longest * top_value)
    return bound, error + steps + 2.0**-22 * lse.abs().nan_to_num(0.0, 0.0, 0.0) + 2.0**-20


# ---------------------------------------------------------------------------
# Pages
# ---------------------------------------------------------------------------


def fork(pools, pages, lengths, refs, parents):
    """New (pages, lengths, refs); the pools are written."""
    S, P = pages.shape
    page = pools[0].shape[1]
    old_pages, old_lengths = pages.tolist(), lengths.tolist()
    free = [i for i, r in enumerate(refs.tolist()) if r == 0]
    count = refs.clone()
    for row in old_pages:
        for at in row:
            if 0 <= at < len(refs):
                count[at] -= 1
    taken, seen, moves = 0, set(), []
    new_pages, new_lengths = [], []
    for s in range(S):
        p = int(parents[s])
        if not 0 <= p < S:
            new_pages.append([-1] * P)
            new_lengths.append(0)
            continue
        row, n = list(old_pages[p]), min(max(old_lengths[p], 0), P * page)
        if n % page and p in seen and 0 <= row[n // page] < len(refs):
            if taken == len(free):
                new_pages.append([-1] * P)
                new_lengths.append(0)
                continue
            moves.append((row[n // page], free[taken], n % page))
            row[n // page] = free[taken]
            taken += 1
        seen.add(p)
        new_pages.append(row)
        new_lengths.append(n)
    for row in new_pages:
        for at in row:
            if 0 <= at < len(refs):
                count[at] += 1
    for a, b, n in moves:
        for pool in pools:
            pool[b, :n] = pool[a, :n]
    return torch.tensor(new_pages, dtype=torch.int32), torch.tensor(new_lengths, dtype=torch.int32), count


def extend(pages, lengths, refs, counts, page):
    S, P = pages.shape
    pages, lengths, refs = pages.clone(), lengths.clone(), refs.clone()
    free = [i for i, r in enumerate(refs.tolist()) if r == 0]
    taken, full = 0, False
    for s in range(S):
        n = min(max(int(lengths[s]), 0), P * page)
        lengths[s] = n
        more = max(int(counts[s]), 0)
        if n + more > P * page:
            continue
        held, wanted = -(-n // page), -(-(n + more) // page)
        full = full or taken + wanted - held > len(free)
        if full and wanted > held:
            continue
        for c in range(held, wanted):
            pages[s, c] = free[taken]
            refs[free[taken]] = 1
            taken += 1
        lengths[s] = n + more
    return pages, lengths, refs


def write(pools, news, pages, lengths, counts):
    S, N = news[0].shape[:2]
    page = pools[0].shape[1]
    for s in range(S):
        n = min(max(int(lengths[s]), 0), pages.shape[1] * page)
        count = min(N if counts is None else max(int(counts[s]), 0), N, n)
        for j in range(count):
            t = n - count + j
            entry = int(pages[s, t // page])
            if 0 <= entry < pools[0].shape[0]:
                for pool, new in zip(pools, news, strict=True):
                    pool[entry, t % page] = new[s, j]


def keep_tokens(pools, pages, lengths, refs, drafted, keep, kept):
    page = pools[0].shape[1]
    pages, refs = pages.clone(), refs.clone()
    out = []
    for s in range(pages.shape[0]):
        n = min(max(int(lengths[s]), 0), pages.shape[1] * page)
        draft = min(max(int(drafted[s]), 0), n)
        line, last = [], -1
        for i in range(min(max(int(kept[s]), 0), keep.shape[1], draft)):
            node = int(keep[s, i])
            if node <= last or node >= draft:
                break
            line.append(node)
            last = node
        start = n - draft
        for pool in pools:
            rows = [pool[int(pages[s, (start + node) // page]), (start + node) % page].clone() for node in line]
            for i, row in enumerate(rows):
                pool[int(pages[s, (start + i) // page]), (start + i) % page] = row
        out.append(start + len(line))
        for c in range(-(-out[-1] // page), pages.shape[1]):
            if 0 <= int(pages[s, c]) < len(refs):
                refs[int(pages[s, c])] -= 1
            pages[s, c] = -1
    return pages, torch.tensor(out, dtype=torch.int32), refs


def reorder(state, parents):
    out = torch.zeros_like(state)
    for b in range(parents.shape[0]):
        for k in range(parents.shape[1]):
            p = int(parents[b, k])
            if 0 <= p < parents.shape[1]:
                out[b, k] = state[b, p]
    return out


def reorder_gradient(grad, parents):
    """In float64, and the sums of the terms' magnitudes."""
    out, size = torch.zeros_like(grad, dtype=torch.float64), torch.zeros_like(grad, dtype=torch.float64)
    for b in range(parents.shape[0]):
        for k in range(parents.shape[1]):
            p = int(parents[b, k])
            if 0 <= p < parents.shape[1]:
                out[b, p] += grad[b, k].double()
                size[b, p] += grad[b, k].double().abs()
    return out, size
