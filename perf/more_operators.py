# SPDX-License-Identifier: MIT
"""More operators of a model in a beam search, as cases that a timing program can
list, draw, prepare, run and check: log-probabilities of given tokens, rotary
positions, and the eviction of cached tokens by the attention that they got.

A case is a dict of plain values; ``kind`` says what runs:

* ``score``: :func:`beamgrad_amd.token_logprobs` of ``[B, T, V]`` logits;
  ``top``: alternatives that are returned; ``entropy``: returned too;
  ``ragged``: sequences end early, their tokens -1 from there on; ``banned``: a
  hundredth of the vocabulary is masked; ``train``: the logits' gradient too.
* ``rotary``: :func:`beamgrad_amd.rotary` of queries ``[S, N, H, D]`` and keys
  ``[S, N, Hkv, D]``; ``width``: values of a head that turn; ``far``: the largest
  position; ``factor``: positions are stretched by it; ``mode``: ``new``,
  ``inplace``, or ``train`` (new tensors and the gradients).
* ``weigh``: :func:`beamgrad_amd.accumulate_weights`: the attention of ``N`` tokens at the
  end of each of ``S`` sequences of ``lo`` to ``hi`` cached ones ahead, summed up for each
  cached token; ``tree``: these are a drafted tree; ``ragged``: from 1 to ``N`` of them ask;
  ``idle``: slots of the batch without a sequence.
* ``evict``: :func:`beamgrad_amd.evict_tokens`: of ``lo`` to ``hi`` tokens of each of
  ``S`` sequences, ``budget`` stay, in ``layers`` layers of keys and values;
  ``joint``: all heads of a layer keep the same ones.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _score(dtype, B, T, V, top=0, entropy=False, ragged=False, banned=False, train=False):
    return dict(kind="score", dtype=dtype, B=B, T=T, V=V, top=top, entropy=entropy, ragged=ragged, banned=banned, train=train)


def _rotary(dtype, S, N, H, Hkv, D, width, interleaved, far, mode, factor=1.0):
    return dict(kind="rotary", dtype=dtype, S=S, N=N, H=H, Hkv=Hkv, D=D, width=width, interleaved=interleaved, far=far,
                mode=mode, factor=factor)


def _weigh(dtype, S, N, H, Hkv, D, page, lo, hi, tree=False, ragged=False, idle=0):
    return dict(kind="weigh", dtype=dtype, S=S, N=N, H=H, Hkv=Hkv, D=D, page=page, lo=lo, hi=hi, tree=tree, ragged=ragged,
                idle=idle)


def _evict(dtype, S, layers, Hkv, D, page, lo, hi, budget, recent, first, joint=False):
    return dict(kind="evict", dtype=dtype, S=S, layers=layers, Hkv=Hkv, D=D, page=page, lo=lo, hi=hi, budget=budget,
                recent=recent, first=first, joint=joint)


def listed():
    cases = {
        # The four beams of one small search, their alternatives shown: latency.
        "score beams f32": _score("float32", 1, 4, 32000, top=5, entropy=True),
        # A step of a serving batch whose users ask for alternatives.
        "score served bf16": _score("bfloat16", 32, 1, 151936, top=20, entropy=True),
        # The beams of a search scored again with a gradient, as minimum-risk training does.
        "rescore trained bf16": _score("bfloat16", 128, 32, 128256, ragged=True, train=True),
        # An odd vocabulary with masked entries, trained on the entropy and the alternatives too.
        "entropy trained f16": _score("float16", 20, 33, 50257, top=4, entropy=True, ragged=True, banned=True, train=True),
        # One token of each sequence of a serving batch, at far positions: latency.
        "rotary step bf16": _rotary("bfloat16", 32, 1, 32, 8, 128, 128, False, 131000, "inplace"),
        # A training step's queries and keys.
        "rotary trained bf16": _rotary("bfloat16", 4, 4096, 32, 8, 128, 128, False, 4096, "train"),
        # Neighbours that turn, in a part of an odd head, in 32 bits, stretched for a long context.
        "rotary part f32": _rotary("float32", 3, 701, 15, 5, 72, 40, True, 30000, "new", factor=4.0),
        # A step of a serving batch, every cached token weighed.
        "weigh tokens bf16": _weigh("bfloat16", 32, 1, 32, 8, 128, 16, 2000, 16000),
        # The ends of two long prompts weigh what came before them.
        "weigh prompts bf16": _weigh("bfloat16", 2, 512, 32, 8, 128, 32, 4000, 16000),
        # Drafted trees of a small batch, an idle slot in it.
        "weigh trees f16": _weigh("float16", 6, 45, 12, 4, 72, 24, 300, 2700, tree=True, ragged=True, idle=1),
        # One sequence of a small model, an odd page: latency.
        "evict one f32": _evict("float32", 1, 2, 5, 72, 24, 900, 900, 500, 64, 4),
        # The prompts of a batch cut to half in every layer, each head for itself.
        "evict prompts bf16": _evict("bfloat16", 8, 16, 8, 128, 16, 4500, 8000, 4096, 128, 4),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """An integer of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["score", "score", "rotary", "weigh", "weigh", "evict"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "score":
        V = _spread(rng, 30, 160000)
        top = rng.choice([0, 0, _spread(rng, 1, min(V, 40))])
        rows = _spread(rng, 1, max(1, min(20000, (80_000_000 if top else 250_000_000) // V)))
        B = _spread(rng, 1, rows)
        return _score(dtype, B, rows // B, V, top, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.5)
    Hkv, G = _spread(rng, 1, 16), _spread(rng, 1, 8)
    D = 8 * _spread(rng, 4, 32)
    if kind == "rotary":
        S, mode = _spread(rng, 1, 64), rng.choice(["new", "inplace", "train"])
        N = _spread(rng, 1, max(1, min(4096, 80_000_000 // (S * Hkv * (G + 1) * D))))
        width = rng.choice([D, D, 2 * _spread(rng, 4, D // 2)])
        return _rotary(dtype, S, N, Hkv * G, Hkv, D, width, rng.random() < 0.5, N + _spread(rng, 1, 500000), mode,
                       rng.choice([1.0, 1.0, 8.0]))
    page = rng.choice([8, 16, 16, 20, 32, 48, 64, 128])
    if kind == "weigh":
        form = rng.choice(["token", "tree", "chunk"])
        N = {"token": 1, "tree": _spread(rng, 2, 100), "chunk": _spread(rng, 16, 512)}[form]
        S = _spread(rng, 1, 48 if form != "chunk" else 4)
        hi = _spread(rng, 1, 131000)
        hi = max(1, min(hi, 500_000_000 // (S * Hkv * D * _SIZE[dtype]), 250_000_000 // (S * Hkv * G * N)))
        return _weigh(dtype, S, N, Hkv * G, Hkv, D, page, _spread(rng, 1, hi), hi, form == "tree",
                      form != "token" and rng.random() < 0.5, int(S > 2 and rng.random() < 0.4))
    S, layers = _spread(rng, 1, 16), _spread(rng, 1, 16)
    hi = _spread(rng, 20, 30000)
    hi = max(20, min(hi, 1_000_000_000 // (S * layers * Hkv * D * _SIZE[dtype])))
    budget = _spread(rng, 2, hi)
    recent = _spread(rng, 1, budget)
    return _evict(dtype, S, layers, Hkv, D, page, _spread(rng, 1, hi), hi, budget, recent - 1, min(4, budget - recent),
                  rng.random() < 0.3)


def _spaced(n, lo, hi):
    """n whole numbers of [lo, hi], evenly spread, in no order."""
    return [lo + int(math.modf((i + 0.5) * 0.6180339887498949)[0] * (hi - lo + 1)) for i in range(n)]


def _tokens_of(case):
    """How many tokens each sequence of a ``score`` case has."""
    return _spaced(case["B"], (case["T"] + 1) // 2, case["T"]) if case["ragged"] else [case["T"]] * case["B"]


def _lengths(case):
    """Tokens ahead of the asking ones, and the asking ones, of each sequence of a
    ``weigh`` case; the idle slots hold nothing."""
    S, N = case["S"], case["N"]
    ahead = _spaced(S, case["lo"], case["hi"])
    asking = _spaced(S, 1, N) if case["ragged"] else [N] * S
    for i in range(case["idle"]):
        ahead[(2 * i + 1) % S], asking[(2 * i + 1) % S] = 0, 0
    return ahead, asking


def _tree_parents(case, seed):
    """A drafted tree for each sequence: a few first guesses, each node among
    the children of a recent one."""
    rng = np.random.default_rng([seed, case["N"], case["S"]])
    S, N = case["S"], case["N"]
    at = np.arange(N)
    low = np.maximum(0, at // 2 - 2)
    parents = low + (rng.random((S, N)) * np.maximum(at - low, 1)).astype(np.int64)
    return np.where((at < 3) | (parents >= at), -1, parents).astype(np.int32)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, dtype, g):
    return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_score(case, seed):
    B, T, V = case["B"], case["T"], case["V"]
    g, dtype = _generator(seed), _TORCH[case["dtype"]]
    logits = _randn(B, T, V, dtype=dtype, g=g).mul_(3.0)
    # a few tokens are likely everywhere
    logits += (8.0 / torch.arange(1, V + 1, device="cuda").float().sqrt())[torch.randperm(V, device="cuda", generator=g)].to(dtype)
    if case["banned"]:
        logits.masked_fill_(torch.rand(V, device="cuda", generator=g) < 0.01, float("-inf"))
    # what a model picks is among the likelier of a few
    some = torch.randint(0, V, (B, T, 8), device="cuda", generator=g)
    tokens = some.gather(2, logits.gather(2, some).argmax(2, keepdim=True)).squeeze(2)
    tokens.masked_fill_(torch.arange(T, device="cuda") >= _int(_tokens_of(case))[:, None], -1)
    state = dict(logits=logits, tokens=tokens)
    if case["train"]:
        logits.requires_grad_(True)
        state["grads"] = [torch.randn(B, T, device="cuda", generator=g)]
        if case["entropy"]:
            state["grads"].append(torch.randn(B, T, device="cuda", generator=g) * 0.1)
        if case["top"]:
            state["grads"].append(torch.randn(B, T, case["top"], device="cuda", generator=g) * 0.1)
    return state


def _frequencies(case):
    half = case["width"] // 2
    return 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half) / case["factor"]


def _prepare_rotary(case, seed):
    S, N, D = case["S"], case["N"], case["D"]
    g, dtype = _generator(seed), _TORCH[case["dtype"]]
    first = torch.tensor(_spaced(S, 0, case["far"] - N), device="cuda")
    state = dict(heads=[_randn(S, N, case[h], D, dtype=dtype, g=g) for h in ("H", "Hkv")],
                 positions=first[:, None] + torch.arange(N, device="cuda"), frequencies=_frequencies(case))
    if case["mode"] == "train":
        for t in state["heads"]:
            t.requires_grad_(True)
        state["grads"] = [_randn(S, N, case[h], D, dtype=dtype, g=g) for h in ("H", "Hkv")]
    return state


def _table(lengths, page, seed):
    """A page table of sequences of these lengths, their pages in no order."""
    held = [-(-n // page) for n in lengths]
    place = np.random.default_rng([seed, sum(held)]).permutation(sum(held) + 3).astype(np.int32)
    table = np.full((len(lengths), max(held) + 1), -1, np.int32)
    refs = np.zeros(len(place), np.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = place[at:at + n]
        refs[table[s, :n]] = 1
        at += n
    return torch.from_numpy(table).cuda(), _int(lengths), torch.from_numpy(refs).cuda()


def _prepare_weigh(case, seed):
    S, N, H, Hkv, D, page = (case[k] for k in ("S", "N", "H", "Hkv", "D", "page"))
    ahead, asking = _lengths(case)
    g, dtype = _generator(seed), _TORCH[case["dtype"]]
    table = _table([a + n for a, n in zip(ahead, asking, strict=True)], page, seed)
    state = dict(table=table, k=_randn(len(table[2]), page, Hkv, D, dtype=dtype, g=g),
                 q=_randn(S, N, H, D, dtype=dtype, g=g) * 1.5,
                 weights=torch.rand(S, Hkv, table[0].shape[1] * page, device="cuda", generator=g),
                 counts=_int(asking) if case["ragged"] or case["idle"] else None,
                 parents=torch.from_numpy(_tree_parents(case, seed)).cuda() if case["tree"] else None)
    # what the attention of these tokens left beside its output
    state["lse"] = torch.full((S, N, H), -math.inf, device="cuda")
    for s in range(S):
        if asking[s]:
            state["lse"][s, :asking[s]] = torch.logsumexp(_scores(case, state, s, ahead[s], asking[s], torch.float32), -1).permute(2, 0, 1).flatten(1)
    return state


def _scores(case, state, s, ahead, asking, dtype):
    """``[Hkv, G, asking, tokens]``: the scores of one sequence's asking tokens, -inf where one sees nothing."""
    page, n = case["page"], ahead + asking
    held = state["table"][0][s, :-(-n // page)].long()
    keys = state["k"][held].flatten(0, 1)[:n].to(dtype).permute(1, 2, 0).contiguous()
    q = state["q"][s, :asking].to(dtype).unflatten(1, (case["Hkv"], -1)).permute(1, 2, 0, 3).contiguous()
    score = torch.matmul(q.flatten(1, 2), keys).unflatten(1, q.shape[1:3]).div_(math.sqrt(case["D"]))
    hidden = np.zeros((asking, n), bool)
    parents = state["parents"][s].tolist() if case["tree"] else None
    for i in range(asking):
        hidden[i, ahead + (0 if case["tree"] else i + 1):] = True
        at = i
        while case["tree"] and at >= 0:
            hidden[i, ahead + at] = False
            at = parents[at]
    return score.masked_fill_(torch.from_numpy(hidden).cuda(), -math.inf)


def _prepare_evict(case, seed):
    S, layers, Hkv, D, page = (case[k] for k in ("S", "layers", "Hkv", "D", "page"))
    lengths = _spaced(S, case["lo"], case["hi"])
    table = _table(lengths, page, seed)
    g = _generator(seed)
    stack = _randn(layers, 2, len(table[2]), page, Hkv, D, dtype=_TORCH[case["dtype"]], g=g)
    # a few tokens get most of the attention, some got none
    T = table[0].shape[1] * page
    weights = torch.randn(layers, S, 1 if case["joint"] else Hkv, T, device="cuda", generator=g).mul_(2.0).exp_()
    weights.mul_((torch.rand(weights.shape, device="cuda", generator=g) < 0.97).float())
    weights.mul_((torch.arange(T, device="cuda") < table[1][:, None]).float()[:, None])
    return dict(stack=stack, pools=[p for layer in stack for p in layer], weights=weights, each=list(weights), table=table)


_PREPARE = {"score": _prepare_score, "rotary": _prepare_rotary, "weigh": _prepare_weigh, "evict": _prepare_evict}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, seed), case=case)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _plain_score(s):
    case = s["case"]
    x = s["logits"].detach().float()
    there = s["tokens"] >= 0
    tokens = s["tokens"].clamp(min=0)[..., None]
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    logp = x.sub_(total.log())
    p = e.div_(total)
    out = [torch.where(there, logp.gather(-1, tokens).squeeze(-1), 0.0)]
    entropy = places = None
    if case["entropy"]:
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
        out.append(torch.where(there, entropy, 0.0))
    if case["top"]:
        # one whole number for a value and its place: the largest, of equal ones the first
        bits = s["logits"].detach().float().add_(0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2**32 - torch.arange(case["V"], device="cuda")
        places = order.topk(case["top"], -1).indices
        del bits, order
        out += [torch.where(there[..., None], logp.gather(-1, places), float("-inf")),
                torch.where(there[..., None], places, -1)]
    if case["train"]:
        g = [torch.where(there.reshape(*there.shape, *[1] * (t.dim() - 2)), t, 0.0) for t in s["grads"]]
        sums = g[0]
        if case["top"]:
            sums = sums + g[-1].sum(-1)
        inner = sums[..., None]
        if case["entropy"]:
            inner = inner + g[1][..., None] * torch.where(p > 0, logp + entropy[..., None], 0.0)
        grad = p.mul_(inner).neg_()
        grad.scatter_add_(-1, tokens, g[0][..., None])
        if case["top"]:
            grad.scatter_add_(-1, places, g[-1])
        out.append(grad.to(s["logits"].dtype))
    return out


def _plain_turned(x, angles, case, sign):
    """``[S, N, heads, D]`` with the first ``width`` values of each head turned."""
    half = case["width"] // 2
    cos, sin = angles.cos().float()[:, :, None], (sign * angles.sin()).float()[:, :, None]
    turn, rest = x.detach().float().split((case["width"], case["D"] - case["width"]), -1)
    a, b = (turn[..., 0::2], turn[..., 1::2]) if case["interleaved"] else (turn[..., :half], turn[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    turn = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turn, rest), -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    angles = s["positions"].double()[..., None] * s["frequencies"]
    out = [_plain_turned(x, angles, case, 1.0) for x in s["heads"]]
    if case["mode"] == "inplace":
        for x, y in zip(s["heads"], out, strict=True):
            x.copy_(y)
        return s["heads"]
    if case["mode"] == "train":
        out += [_plain_turned(x, angles, case, -1.0) for x in s["grads"]]
    return out


def _closure(link, doublings):
    """Which nodes are reached over any number of links."""
    if doublings == 0:
        return link > 0
    return _closure((torch.matmul(link, link) > 0).float(), doublings - 1)


def _plain_weigh(s):
    case, (pages, lengths, _refs) = s["case"], s["table"]
    S, N, H, D = s["q"].shape
    Hkv, page = case["Hkv"], case["page"]
    G, L = H // Hkv, pages.shape[1] * page
    counts = torch.full_like(lengths, N) if s["counts"] is None else s["counts"]
    prefix = (lengths - counts).long()
    k = s["k"][pages.clamp(min=0).long()].reshape(S, L, Hkv, D).permute(0, 2, 3, 1).float()
    q = s["q"].reshape(S, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, N * G, D).float()
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).reshape(S, Hkv, N, G, L)
    del k
    node = torch.arange(N, device="cuda")
    if s["parents"] is None:
        sees = (node <= node[:, None]).expand(S, N, N)
    else:
        link = torch.eye(N, device="cuda") + torch.nn.functional.one_hot(s["parents"].long() + 1, N + 1)[..., 1:]
        sees = _closure(link, math.ceil(math.log2(N)))
    j = torch.arange(L, device="cuda") - prefix[:, None]  # [S, L]: the asking token at each place, or one before or after
    asking = (j >= 0) & (j < counts[:, None])
    visible = sees.gather(2, j.clamp(0, N - 1)[:, None, :].expand(S, N, L)) & asking[:, None] | (j < 0)[:, None]
    visible = visible & (node < counts[:, None])[..., None]  # [S, N, L]
    lse = s["lse"].reshape(S, N, Hkv, G).permute(0, 2, 1, 3)[..., None]
    scores.sub_(torch.where(lse == float("-inf"), 0.0, lse)).exp_()
    more = scores.masked_fill_(~visible[:, None, :, None], 0.0).sum((2, 3))
    # those that ask now have no weight yet
    weights = s["weights"]
    weights.copy_(torch.where(asking[:, None], more, torch.where((j < 0)[:, None], weights + more, weights)))
    return [weights]


def _plain_evict(s):
    case, (pages, lengths, refs) = s["case"], s["table"]
    page, budget = case["page"], case["budget"]
    layers, S, heads, T = s["weights"].shape
    at = torch.arange(T, device="cuda")
    n = lengths[:, None]
    recent = min(case["recent"], budget)
    first = min(case["first"], budget - recent)
    sure = (at < first) | (at >= n - recent)
    rank = torch.where(sure[:, None], float("inf"), s["weights"]).masked_fill((at >= n)[:, None], float("-inf"))
    rank = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget].sort(-1).values  # [layers, S, heads, budget]
    over = lengths > budget
    column = torch.arange(rank.shape[-1], device="cuda")
    weights = torch.zeros_like(s["weights"])
    weights[..., :rank.shape[-1]] = s["weights"].gather(-1, rank)
    weights = torch.where(over[:, None, None], weights, s["weights"])
    who = over.nonzero().squeeze(1)
    rank = rank[:, who]
    if case["joint"]:
        rank = rank.expand(-1, -1, case["Hkv"], -1)
    l = torch.arange(layers, device="cuda")[:, None, None, None]
    h = torch.arange(case["Hkv"], device="cuda")[:, None]
    w = who[:, None, None]
    moved = s["stack"][l, :, pages[w, rank // page].long(), rank % page, h]
    s["stack"][l, :, pages[w, column // page].long(), column % page, h] = moved
    lengths = lengths.clamp(max=budget)
    lengths = torch.where(over, lengths, s["table"][1])
    kept = torch.where(torch.arange(pages.shape[1], device="cuda") < -(-lengths // page)[:, None], pages, -1)
    gone = (pages >= 0) & (kept < 0)
    refs = refs.clone().index_add_(0, pages.clamp(min=0).flatten().long(), -gone.flatten().int())
    return [s["stack"], kept, lengths, refs, *weights]


_PLAIN = {"score": _plain_score, "rotary": _plain_rotary, "weigh": _plain_weigh, "evict": _plain_evict}


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------


def _own_score(s):
    import beamgrad_amd as bg

    got = bg.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"], entropy=s["case"]["entropy"])
    out = [t for t in got if t is not None]
    if not s["case"]["train"]:
        return out
    floats = [t for t in out if t.is_floating_point()]
    grad, = torch.autograd.grad(floats, [s["logits"]], s["grads"])
    return [*out, grad]


def _own_rotary(s):
    import beamgrad_amd as bg

    case = s["case"]
    out = bg.rotary(s["heads"], s["positions"], s["frequencies"], interleaved=case["interleaved"],
                    inplace=case["mode"] == "inplace")
    if case["mode"] == "train":
        return [*out, *torch.autograd.grad(out, s["heads"], s["grads"])]
    return out


def _own_weigh(s):
    import beamgrad_amd as bg

    bg.accumulate_weights(s["weights"], s["q"], s["k"], s["lse"], bg.PageTable(*s["table"]), parents=s["parents"],
                          counts=s["counts"])
    return [s["weights"]]


def _own_evict(s):
    import beamgrad_amd as bg

    case = s["case"]
    table, weights = bg.evict_tokens(s["pools"], s["each"], bg.PageTable(*s["table"]), case["budget"], recent=case["recent"],
                                     first=case["first"])
    return [s["stack"], *table, *weights]


_OWN = {"score": _own_score, "rotary": _own_rotary, "weigh": _own_weigh, "evict": _own_evict}


def run(state):
    return list((_OWN if own else _PLAIN)[state["case"]["kind"]](state))


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _pairs(case):
    """Keys that the asking tokens of all sequences see, and cached tokens."""
    ahead, asking = _lengths(case)
    parents = _tree_parents(case, 0) if case["tree"] else None
    pairs = 0
    for s, n in enumerate(asking):
        depth = []
        for i in range(n):
            depth.append(i + 1 if parents is None else 1 + (depth[parents[s, i]] if parents[s, i] >= 0 else 0))
        pairs += n * ahead[s] + sum(depth)
    return pairs, sum(ahead) + sum(asking)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "score":
        rows = sum(_tokens_of(case))  # those of no token need not be read; their gradients are zeros
        small = case["B"] * case["T"] * (8 + 4 + 4 * case["entropy"] + 12 * case["top"])
        back = (rows + case["B"] * case["T"]) * case["V"] * size if case["train"] else 0
        # the largest, the sums, the exponentials
        return {"bytes": rows * case["V"] * size + back + small, "flops": rows * case["V"] * (8 if case["train"] else 4)}
    if case["kind"] == "rotary":
        tokens = case["S"] * case["N"]
        values = tokens * (case["H"] + case["Hkv"])
        passes = 2 if case["mode"] == "train" else 1
        each = case["width"] if case["mode"] == "inplace" else case["D"]
        return {"bytes": passes * (2 * values * each * size + 8 * tokens), "flops": passes * 3 * values * case["width"]}
    if case["kind"] == "weigh":
        pairs, tokens = _pairs(case)
        queries = sum(_lengths(case)[1]) * case["H"]
        return {"bytes": tokens * case["Hkv"] * (case["D"] * size + 8) + queries * (case["D"] * size + 4),
                "flops": pairs * case["H"] * (2 * case["D"] + 3)}
    lengths = [n for n in _spaced(case["S"], case["lo"], case["hi"]) if n > case["budget"]]
    heads = 1 if case["joint"] else case["Hkv"]
    # of the tokens that stay, those ahead of the first that goes need not move; on average few
    moved = len(lengths) * max(0, case["budget"] - case["first"])
    table = 4 * case["S"] * (2 * -(-case["hi"] // case["page"]) + 4)
    return {"bytes": case["layers"] * (4 * moved * case["Hkv"] * case["D"] * size + 4 * heads * (sum(lengths) + case["S"] * case["budget"])) + table,
            "flops": 0}


# ---------------------------------------------------------------------------
# The results by the definitions, one row, sequence or head after the other
# ---------------------------------------------------------------------------


def _exact_score(case, seed):
    s = _prepare_score(case, seed)
    B, T, V = s["logits"].shape
    top = case["top"]
    f64 = dict(dtype=torch.float64, device="cuda")
    lp, entropy = torch.zeros(B, T, **f64), torch.zeros(B, T, **f64)
    best, which = torch.full((B, T, top), -math.inf, **f64), torch.full((B, T, top), -1, device="cuda")
    grad = torch.zeros(B, T, V, **f64) if case["train"] else None
    for b, n in enumerate(_tokens_of(case)):
        if n == 0:
            continue
        x = s["logits"][b, :n].detach().double()
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        at = s["tokens"][b, :n, None]
        lp[b, :n] = logp.gather(1, at)[:, 0]
        h = -torch.special.xlogy(p, p).sum(-1)
        entropy[b, :n] = h
        if top:
            which[b, :n] = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
            best[b, :n] = logp.gather(1, which[b, :n])
        if case["train"]:
            g = [t[b, :n].double() for t in s["grads"]]
            # d log p_t / d x = e_t - p; d H / d x_v = -p_v (log p_v + H)
            row = torch.zeros_like(x).scatter_add_(1, at, g[0][:, None]) - p * g[0][:, None]
            if case["entropy"]:
                row -= g[1][:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
            if top:
                row += torch.zeros_like(x).scatter_add_(1, which[b, :n], g[-1]) - p * g[-1].sum(-1, keepdim=True)
            grad[b, :n] = row
    out = [lp]
    out += [entropy] if case["entropy"] else []
    out += [best, which] if top else []
    return out + ([grad] if case["train"] else [])


def _exact_rotary(case, seed):
    s = _prepare_rotary(case, seed)
    half = case["width"] // 2
    at = torch.arange(half, device="cuda")
    first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + half)
    unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[..., None] * s["frequencies"])[:, :, None]

    def turned(x, by):
        out = x.detach().double()
        pair = torch.complex(out[..., first], out[..., second]) * by
        out[..., first], out[..., second] = pair.real, pair.imag
        return out

    return [turned(x, unit) for x in s["heads"]] + [turned(x, unit.conj()) for x in s.get("grads", ())]


def _exact_weigh(case, seed):
    s = _prepare_weigh(case, seed)
    out = s["weights"].double()
    for b, (ahead, n) in enumerate(zip(*_lengths(case), strict=True)):
        if n == 0:
            continue
        lse = s["lse"][b, :n].double().unflatten(1, (case["Hkv"], -1)).permute(1, 2, 0)[..., None]
        more = (_scores(case, s, b, ahead, n, torch.float64) - lse).exp_().sum((1, 2))
        out[b, :, :ahead] += more[:, :ahead]
        out[b, :, ahead:ahead + n] = more[:, ahead:]
    return [out]


def _exact_evict(case, seed):
    s = _prepare_evict(case, seed)
    pages, lengths, refs = (t.cpu().numpy() for t in s["table"])
    page, budget = case["page"], case["budget"]
    stack, out = s["stack"], torch.zeros_like(s["weights"])
    weights = s["weights"].cpu().numpy()
    new_pages, new_lengths, new_refs = pages.copy(), lengths.copy(), refs.copy()
    for b, n in enumerate(lengths.tolist()):
        if n <= budget:
            out[:, b] = s["weights"][:, b]
            continue
        recent = min(case["recent"], budget)
        first = min(case["first"], budget - recent)
        place = lambda j, b=b: (torch.from_numpy(pages[b, j // page]).long().cuda(), torch.from_numpy(j % page).cuda())  # noqa: E731
        for layer in range(case["layers"]):
            for h in range(weights.shape[2]):
                middle = np.arange(first, n - recent)
                best = middle[np.lexsort((middle, -weights[layer, b, h, middle]))][:budget - recent - first]
                keep = np.concatenate([np.arange(first), np.sort(best), np.arange(n - recent, n)])
                out[layer, b, h, :budget] = s["weights"][layer, b, h, torch.from_numpy(keep).cuda()]
                heads = slice(None) if case["joint"] else slice(h, h + 1)
                for pool in stack[layer]:
                    (fp, fo), (tp, to) = place(keep), place(np.arange(budget))
                    pool[tp, to, heads] = pool[fp, fo, heads]
        held = -(-budget // page)
        for at in pages[b, held:]:
            if at >= 0:
                new_refs[at] -= 1
        new_pages[b, held:] = -1
        new_lengths[b] = budget
    return [stack, *(torch.from_numpy(t).cuda() for t in (new_pages, new_lengths, new_refs)), *out]


_EXACT = {"score": _exact_score, "rotary": _exact_rotary, "weigh": _exact_weigh, "evict": _exact_evict}


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)
