# SPDX-License-Identifier: MIT
"""Plain restatements, in 64 bits on the CPU, of log-probabilities of given tokens,
rotary positions, the attention that cached tokens get, and the eviction by it;
with how far 32-bit arithmetic may take a kernel from them."""

from __future__ import annotations

import math

import torch

from tests.paged_reference import HALF_STEP, seen_by

STEP = 2.0**-24  # half a step of float32


def token_logprobs(logits, tokens, top, entropy, grads=None):
    """A dict of the results, and with ``grads`` (of log-probabilities, entropy,
    alternatives; None: zeros) the logits' gradient; and a dict of bounds.

    Bounds. A row's exponentials are within (2 |d| + 4) half steps of theirs, d being
    the distance to the maximum (its rounding, that of its product with log2(e),
    and the exponential's own); weighted by the probabilities that is 2 E + 4, E = the
    sum of p |d|, at most the largest |log p| weighted. A thread adds up to V / 64 of
    them and their rescalings, and 20 more joins: s is within (V / 64 + 2 E + 24 + 16)
    half steps, and so, in absolute terms, is log s; the two subtractions of log p
    and the logarithm add 3 half steps of their values."""
    shape, V = tuple(tokens.shape), logits.shape[-1]
    x, t = logits.reshape(-1, V).double(), tokens.reshape(-1).long()
    rows = x.shape[0]
    lp, h = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    best, which = torch.full((rows, top), -math.inf, dtype=torch.float64), torch.full((rows, top), -1)
    grad, grad_bound = torch.zeros(rows, V, dtype=torch.float64), torch.zeros(rows, V, dtype=torch.float64)
    lp_bound, h_bound, best_bound = torch.zeros_like(lp), torch.zeros_like(lp), torch.zeros_like(best)
    half = HALF_STEP[logits.dtype]
    flat = [None if g is None else g.reshape(rows, *g.shape[len(shape):]).double() for g in grads or (None, None, None)]
    for r in range(rows):
        if not 0 <= int(t[r]) < V:
            continue
        row = x[r]
        if row.isnan().any() or (row == math.inf).any():
            lp[r] = h[r] = math.nan
            best[r] = math.nan
            grad[r] = math.nan
            continue
        order = torch.sort(row, descending=True, stable=True).indices[:top]
        which[r] = order
        if (row == -math.inf).all():
            lp[r] = -math.inf
            continue
        logp = torch.log_softmax(row, 0)
        p = logp.exp()
        some = torch.where(p > 0, logp, 0.0)
        lp[r], best[r], h[r] = logp[t[r]], logp[order], -(p * some).sum()
        spread = float((p * (row.max() - row).nan_to_num(0.0, 0.0, 0.0)).sum())
        of_sum = STEP * (V / 64 + 2 * spread + 40)
        distance = (row - row.max()).abs().nan_to_num(0.0, 0.0, 0.0)
        of_logp = of_sum + STEP * (distance + 3 * some.abs() + 3)
        lp_bound[r], best_bound[r] = of_logp[t[r]], of_logp[order]
        h_bound[r] = of_sum * (2 + 2 * spread) + STEP * 4 * (1 + spread)
        g, g_h, g_top = (None if f is None else f[r] for f in flat)
        total = (0.0 if g is None else float(g)) + (0.0 if g_top is None else float(g_top.sum()))
        size = (0.0 if g is None else abs(float(g))) + (0.0 if g_top is None else float(g_top.abs().sum()))
        by = 0.0 if g_h is None else float(g_h)
        inner = total + by * torch.where(p > 0, some + h[r], 0.0)
        grad[r] = -p * inner
        # p is within of_logp (and the exponential's 4 half steps); its factor is a sum of
        # up to 66 terms
        magnitude = p * (size + abs(by) * (some.abs() + h[r].abs()))
        grad_bound[r] = magnitude * (of_logp + 80 * STEP) + p * abs(by) * (h_bound[r] + of_logp)
        if g is not None:
            grad[r, t[r]] += g
        if g_top is not None:
            grad[r, order] += g_top
        # what is added at a token is one more sum
        direct = torch.zeros(V, dtype=torch.float64)
        if g is not None:
            direct[t[r]] += g.abs()
        if g_top is not None:
            direct[order] += g_top.abs()
        # (a 16-bit type's least step bounds small values)
        least = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}[logits.dtype]
        grad_bound[r] += direct * (of_logp + 70 * STEP)
        grad_bound[r] = grad_bound[r] * (1 + half) + half * grad[r].abs() + least
    result = dict(logprobs=lp.reshape(shape), entropy=h.reshape(shape) if entropy else None,
                  top_logprobs=best.reshape(*shape, top) if top else None, top_tokens=which.reshape(*shape, top) if top else None,
                  grad=grad.reshape(logits.shape))
    bounds = dict(logprobs=lp_bound.reshape(shape), entropy=h_bound.reshape(shape), top_logprobs=best_bound.reshape(*shape, top),
                  grad=grad_bound.reshape(logits.shape))
    return result, bounds


def rotary(x, positions, frequencies, interleaved, scale, counts=None, inverse=False):
    """``(result, bound)``: a sine or cosine is within 2 half steps of 1 (its sum, its
    argument, the scale), a product and a sum of two round once each."""
    half = frequencies.numel()
    at = torch.arange(half)
    first, second = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
    angle = positions.double()[..., None] * frequencies.double()
    cos, sin = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None] * (-1.0 if inverse else 1.0)
    out, a, b = x.double().clone(), x[..., first].double(), x[..., second].double()
    out[..., first], out[..., second] = scale * (a * cos - b * sin), scale * (a * sin + b * cos)
    bound = torch.zeros_like(out)
    size = (a.abs() + b.abs()) * abs(scale) * 6 * STEP
    bound[..., first], bound[..., second] = size, size
    if counts is not None:
        past = torch.arange(x.shape[1]) >= counts[:, None]
        out[past] = 0.0
        bound[past] = 0.0
    half_step = HALF_STEP[x.dtype]
    least = {torch.float32: 2.0**-140, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}[x.dtype]
    turned = bound > 0
    return out, torch.where(turned, bound * (1 + half_step) + half_step * out.abs() + least, 0.0)


def accumulate(weights, q, k, lse, pages, lengths, counts, parents, scale):
    """``(weights, bound)``. A score is a sum of D products, within (D + 2) half steps of
    the sum of their sizes; with the log-sum's product and the final sum, in units of
    the exponent, each rounding to half a step of its value: the exponential moves by
    that, and by 4 half steps of its own; a key's sum adds one a row, and the old
    weight one more."""
    S, N, H, D = q.shape
    n_pages, page, Hkv, _ = k.shape
    G, P = H // Hkv, pages.shape[1]
    out, bound = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    for s in range(S):
        length = min(max(int(lengths[s]), 0), P * page)
        count = min(max(int(counts[s]), 0), N, length)
        ahead = length - count
        if count == 0:
            continue
        there = [t for t in range(length) if 0 <= int(pages[s, t // page]) < n_pages]
        keys = torch.zeros(length, Hkv, D, dtype=torch.float64)
        for t in there:
            keys[t] = k[int(pages[s, t // page]), t % page].double()
        sums, sizes = torch.zeros(Hkv, length, dtype=torch.float64), torch.zeros(Hkv, length, dtype=torch.float64)
        for i in range(count):
            seen = torch.zeros(length, dtype=torch.bool)
            seen[:ahead] = True
            for j in seen_by(i, count, None if parents is None else parents[s]):
                seen[ahead + j] = True
            for h in range(H):
                l = float(lse[s, i, h])
                if l == -math.inf:
                    continue
                key, row = keys[:, h // G], q[s, i, h].double()
                score = key @ row * scale
                w = torch.where(seen, torch.exp(score - l), 0.0)
                off = STEP * ((D + 2) * (key.abs() @ row.abs()) * scale + 3 * score.abs() + 3 * abs(l) + 4 + (score - l).abs())
                sums[h // G] += w
                sizes[h // G] += w * torch.expm1(off.clamp(max=50.0))
        sizes += sums * STEP * (count * G + 40)
        for t in there:
            if t < ahead:
                out[s, :, t] += sums[:, t]
            else:
                out[s, :, t] = sums[:, t]
            bound[s, :, t] = sizes[:, t] + 2 * STEP * out[s, :, t].abs()
    return out, bound


def evict(pools, weights, pages, lengths, refs, budgets, recent, first):
    """New (pages, lengths, refs, weights); the pools are written."""
    S, P = pages.shape
    page, n_pages = pools[0].shape[1], refs.numel()
    each = len(pools) // len(weights)
    new_pages, new_lengths, new_refs = pages.clone(), lengths.clone(), refs.clone()
    new_weights = [w.clone() for w in weights]
    old = [p.clone() for p in pools]
    for s in range(S):
        n = min(max(int(lengths[s]), 0), P * page)
        new_lengths[s] = n
        b = max(int(budgets[s]), 0)
        if n <= b:
            continue
        r = min(recent, b)
        f = min(first, b - r)
        held, low, high = -(-n // page), f // page, -(-b // page)
        row = pages[s].tolist()
        if any(not 0 <= row[c] < n_pages for c in range(held)) or any(int(refs[row[c]]) != 1 for c in range(low, high)):
            continue
        for i, w in enumerate(weights):
            for g in range(w.shape[1]):
                value = w[s, g].tolist()
                middle = sorted(range(f, n - r), key=lambda t: (-math.inf if math.isnan(value[t]) else value[t], not math.isnan(value[t])),
                                reverse=True)  # (a stable sort keeps equal ones in order, in reverse too)
                keep = [*range(f), *sorted(middle[:b - r - f]), *range(n - r, n)]
                new_weights[i][s, g] = 0.0
                for place, token in enumerate(keep):
                    new_weights[i][s, g, place] = w[s, g, token]
                    for p in range(i * each, (i + 1) * each):
                        heads = slice(None) if w.shape[1] == 1 else slice(g, g + 1)
                        pools[p][row[place // page], place % page][heads] = old[p][row[token // page], token % page][heads]
        for c in range(high, P):
            if 0 <= row[c] < n_pages:
                new_refs[row[c]] -= 1
            new_pages[s, c] = -1
        new_lengths[s] = b
    return new_pages, new_lengths, new_refs, new_weights
