# SPDX-License-Identifier: MIT
"""CPU checks of token log-probabilities, rotary positions, and eviction: what they
refuse, their shapes without a GPU, and what the C entries refuse before a launch."""

import math
import os
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import beamgrad_amd as bg
from beamgrad_amd import _build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
META = torch.device("meta")
I32, I64 = torch.int32, torch.int64


def table(S=4, P=5, n_pages=20, device="cpu"):
    return bg.PageTable.empty(S, P, n_pages, device=device)


def score(logits=None, tokens=None, **more):
    return bg.token_logprobs(torch.zeros(4, 9) if logits is None else logits, torch.zeros(4, dtype=I64) if tokens is None else tokens, **more)


def turn(tensors=None, positions=None, frequencies=None, **more):
    return bg.rotary([torch.zeros(2, 3, 4, 8)] if tensors is None else tensors, torch.zeros(2, 3, dtype=I64) if positions is None else positions,
                     torch.ones(4, dtype=torch.float64) if frequencies is None else frequencies, **more)


def weigh(**change):
    a = dict(weights=torch.zeros(4, 2, 40), q=torch.zeros(4, 3, 4, 16), k=torch.zeros(20, 8, 2, 16), lse=torch.zeros(4, 3, 4), table=table())
    a.update(change)
    w, q, k, lse, t = (a.pop(n) for n in ("weights", "q", "k", "lse", "table"))
    return bg.accumulate_weights(w, q, k, lse, t, **a)


def evict(**change):
    a = dict(pools=[torch.zeros(20, 8, 2, 4) for _ in range(2)], weights=[torch.zeros(4, 2, 40)], table=table(), budget=7)
    a.update(change)
    pools, weights, t, budget = (a.pop(n) for n in ("pools", "weights", "table", "budget"))
    return bg.evict_tokens(pools, weights, t, budget, **a)


def test_accepted_calls_need_the_gpu():
    ones = torch.ones(4, dtype=I32)
    for call in (score, lambda: score(top=9, entropy=True), lambda: score(torch.zeros(9), torch.tensor(1)), turn,
                 lambda: turn(inplace=True, counts=torch.ones(2, dtype=I32), interleaved=True, scale=-2.0),
                 lambda: turn([torch.zeros(2, 3, 1, 9), torch.zeros(2, 3, 5, 64)], frequencies=torch.ones(4)),
                 weigh, lambda: weigh(parents=torch.zeros(4, 3, dtype=I64), counts=ones, scale=0.5), evict,
                 lambda: evict(budget=ones, recent=3, first=1), lambda: evict(weights=[torch.zeros(4, 1, 40) for _ in range(2)])):
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            call()


@pytest.mark.parametrize("change, error, message", [
    (dict(logits=torch.zeros(4, 9, dtype=torch.float64)), ValueError, "float32, float16 or bfloat16"),
    (dict(logits=torch.zeros(4, 0)), ValueError, "must be a .*V"),
    (dict(logits=torch.zeros(())), ValueError, "must be a .*V"),
    (dict(tokens=torch.zeros(3, dtype=I64)), ValueError, "tokens must be an int32 or int64 .4"),
    (dict(tokens=torch.zeros(4, 1, dtype=I64)), ValueError, "tokens must be"),
    (dict(tokens=torch.zeros(4)), ValueError, "tokens must be"),
    (dict(top=10), ValueError, "top must be in .0, 9"),
    (dict(top=-1), ValueError, "top must be in"),
    (dict(logits=torch.zeros(4, 100), top=65), ValueError, "top must be in .0, 64"),
    (dict(top=True), TypeError, "top must be an int"),
    (dict(top=2.0), TypeError, "top must be an int"),
    (dict(logits=[0.0]), TypeError, "logits must be a torch.Tensor"),
    (dict(tokens=[0]), TypeError, "tokens must be a torch.Tensor"),
    (dict(logits=torch.zeros(1, 1).expand(1 << 24, 1), tokens=torch.zeros(1, dtype=I32).expand(1 << 24)), ValueError, "fewer than 2..24 rows"),
])
def test_score_refusals(change, error, message):
    with pytest.raises(error, match=message):
        score(**change)


@pytest.mark.parametrize("change, error, message", [
    (dict(tensors=[torch.zeros(2, 3, 8)]), ValueError, "must be .S, N, H, D"),
    (dict(tensors=[torch.zeros(2, 4, 1, 8)]), ValueError, "must be .S, N, H, D"),
    (dict(tensors=[torch.zeros(2, 3, 0, 8)]), ValueError, "must be .S, N, H, D"),
    (dict(tensors=[torch.zeros(2, 3, 1, 8, dtype=torch.float64)]), ValueError, "float32, float16 or bfloat16"),
    (dict(tensors=[torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 1, 8).half()]), ValueError, "one type"),
    (dict(tensors=[torch.zeros(2, 3, 1, 7)]), ValueError, "from 8 .* wide, got 7"),
    (dict(tensors=[torch.zeros(2, 3, 1, 1025)]), ValueError, "to 1024 wide"),
    (dict(positions=torch.zeros(2, 3)), ValueError, "positions must be"),
    (dict(positions=torch.zeros(6, dtype=I64)), ValueError, "positions must be"),
    (dict(frequencies=torch.ones(4, dtype=I64)), ValueError, "frequencies must be"),
    (dict(frequencies=torch.ones(0)), ValueError, "frequencies must be"),
    (dict(frequencies=torch.ones(2, 2)), ValueError, "frequencies must be"),
    (dict(counts=torch.ones(3, dtype=I32)), ValueError, "counts must be"),
    (dict(scale=math.inf), ValueError, "scale must be finite"),
    (dict(scale=1e300), ValueError, "scale must be finite"),
    (dict(tensors=[torch.zeros(2, 3, 8, 4).transpose(2, 3)], inplace=True), ValueError, "contiguous to be turned in place"),
    (dict(tensors=[[1.0]]), TypeError, "a list in it"),
    (dict(positions=[1]), TypeError, "positions must be a torch.Tensor"),
    (dict(frequencies=torch.ones(4, dtype=torch.float64, requires_grad=True)), RuntimeError, "no gradient of its frequencies"),
    (dict(tensors=[torch.zeros(2, 3, 4, 8, requires_grad=True)], inplace=True), RuntimeError, "no gradient"),
])
def test_rotary_refusals(change, error, message):
    with pytest.raises(error, match=message):
        turn(**change)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("S, N", [(0, 3), (2, 0)])
def test_rotary_of_a_batch_without_tokens_is_checked(S, N, inplace):
    """As any other: it needs the GPU, and heads that fit."""
    at = torch.zeros(S, N, dtype=I64)
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        turn([torch.zeros(S, N, 4, 8)], at, inplace=inplace)
    for bad in ((S, N, 0, 8), (S, N, 4, 7), (S, N, 4, 0), (S, N + 1, 4, 8), (S + 1, N, 4, 8)):
        with pytest.raises(ValueError):
            turn([torch.zeros(bad)], at, inplace=inplace)
    with pytest.raises(ValueError, match="counts must be"):
        turn([torch.zeros(S, N, 4, 8)], at, counts=torch.zeros(S + 1, dtype=I32), inplace=inplace)


def test_frequencies():
    f = bg.rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(bg.rotary_frequencies(8, factor=4.0, device="cpu") * 4, f, rtol=1e-15)
    mixed = bg.rotary_frequencies(64, base=500000.0, factor=8.0, context=8192, device="cpu")
    own = bg.rotary_frequencies(64, base=500000.0, device="cpu")
    turns = 8192 * own / (2 * math.pi)
    assert torch.equal(mixed[turns >= 4], own[turns >= 4]) and torch.equal(mixed[turns <= 1], own[turns <= 1] / 8)
    between = (turns > 1) & (turns < 4)
    part = (turns[between] - 1) / 3
    assert between.any() and torch.allclose(mixed[between], own[between] * (part + (1 - part) / 8), rtol=1e-14)
    for bad in (dict(width=7), dict(width=0), dict(width=8, base=0.0), dict(width=8, factor=-1.0), dict(width=8, context=0),
                dict(width=8, context=5, turns=(2.0, 2.0))):
        with pytest.raises(ValueError):
            bg.rotary_frequencies(bad.pop("width"), device="cpu", **bad)


@pytest.mark.parametrize("change, error, message", [
    (dict(weights=torch.zeros(4, 2, 39)), ValueError, "weights must be a float32 .4, 2, 40"),
    (dict(weights=torch.zeros(4, 4, 40)), ValueError, "weights must be"),
    (dict(weights=torch.zeros(4, 2, 40).half()), ValueError, "weights must be"),
    (dict(weights=torch.zeros(4, 2, 80)[..., ::2]), ValueError, "places must be contiguous"),
    (dict(weights=torch.zeros(1, 2, 40).expand(4, 2, 40)), ValueError, "overlap"),
    (dict(weights=torch.zeros(4, 1, 40).expand(4, 2, 40)), ValueError, "overlap"),
    (dict(weights=torch.zeros(1000).as_strided((4, 2, 40), (40, 40, 1))), ValueError, "overlap"),
    (dict(lse=torch.zeros(4, 3, 2)), ValueError, "lse must be"),
    (dict(lse=torch.zeros(4, 3, 4).double()), ValueError, "lse must be"),
    (dict(q=torch.zeros(4, 3, 3, 16), lse=torch.zeros(4, 3, 3)), ValueError, "multiple of the cache's 2"),
    (dict(k=torch.zeros(20, 8, 2, 16).half()), ValueError, "one type"),
    (dict(k=torch.zeros(20, 8, 2, 17)[..., :16]), ValueError, "multiples of 16 bytes"),
    (dict(scale=0.0), ValueError, "scale must be positive"),
    (dict(counts=torch.ones(4)), ValueError, "counts must be"),
    (dict(parents=torch.ones(4, 2, dtype=I32)), ValueError, "parents must be"),
    (dict(table=tuple(table())), TypeError, "PageTable"),
    (dict(lse=None), TypeError, "lse must be a torch.Tensor"),
    (dict(q=torch.zeros(4, 3, 4, 16, requires_grad=True)), RuntimeError, "no gradient"),
    (dict(weights=torch.zeros(4, 2, 40, requires_grad=True)), RuntimeError, "no gradient"),
])
def test_weight_refusals(change, error, message):
    with pytest.raises(error, match=message):
        weigh(**change)


POOL = torch.zeros(20, 8, 2, 4)


@pytest.mark.parametrize("change, error, message", [
    (dict(pools=[]), ValueError, "at least one pool"),
    (dict(weights=[]), ValueError, "multiple of the weights"),
    (dict(weights=[torch.zeros(4, 2, 40)] * 3), ValueError, "multiple of the weights"),
    (dict(weights=[torch.zeros(4, 40)]), ValueError, "must be .S, heads, places"),
    (dict(weights=[torch.zeros(4, 2, 41)]), ValueError, "weights.0. must be a float32 .4, 2, 40"),
    (dict(weights=[torch.zeros(4, 2, 40), torch.zeros(4, 1, 40)]), ValueError, "weights.1. must be"),
    (dict(weights=[torch.zeros(4, 2, 40).double()]), ValueError, "weights.0. must be"),
    (dict(weights=[torch.zeros(4, 3, 40)]), ValueError, "weights of 3 heads need pools"),
    (dict(pools=[torch.zeros(20, 8, 4)]), ValueError, "weights of 2 heads need pools"),
    (dict(pools=[torch.zeros(19, 8, 2, 4)]), ValueError, "must have 20 pages"),
    (dict(pools=[POOL, POOL]), ValueError, "share memory"),
    (dict(pools=[torch.zeros(1, 8, 2, 4).expand(20, 8, 2, 4)]), ValueError, "overlap"),
    (dict(budget=-1), ValueError, "budget must be in"),
    (dict(budget=2**31), ValueError, "budget must be in"),
    (dict(budget=torch.ones(3, dtype=I32)), ValueError, "budget must be an int32"),
    (dict(budget=torch.ones(4)), ValueError, "budget must be an int32"),
    (dict(recent=-1), ValueError, "recent must be in"),
    (dict(first=2**31), ValueError, "first must be in"),
    (dict(weights=[[0.0]]), TypeError, "weights must be a sequence of tensors"),
    (dict(pools=[torch.zeros(20, 8, 2, 4, requires_grad=True)], weights=[torch.zeros(4, 2, 40)]), RuntimeError, "no gradient"),
    (dict(weights=[torch.zeros(4, 2, 40, requires_grad=True)]), RuntimeError, "no gradient"),
])
def test_evict_refusals(change, error, message):
    with pytest.raises(error, match=message):
        evict(**change)


def test_shapes_without_a_gpu():
    """Meta and fake tensors, their gradients too."""
    def calls(zeros, device):
        logits = zeros(2, 3, 50).requires_grad_()
        got = bg.token_logprobs(logits, zeros(2, 3, dtype=I64), top=4, entropy=True)
        assert [t.shape for t in got] == [(2, 3), (2, 3), (2, 3, 4), (2, 3, 4)] and got.top_tokens.dtype == I64
        assert [t.requires_grad for t in got] == [True, True, True, False]
        grad, = torch.autograd.grad([got.logprobs.sum() + got.entropy.sum()], logits)
        assert grad.shape == logits.shape
        x = zeros(2, 3, 4, 8).requires_grad_()
        out = bg.rotary([x, zeros(2, 3, 1, 9)], zeros(2, 3, dtype=I64), zeros(4, dtype=torch.float64))
        assert [t.shape for t in out] == [(2, 3, 4, 8), (2, 3, 1, 9)] and not out[1].requires_grad
        assert torch.autograd.grad(out[0].sum(), x)[0].shape == x.shape
        assert bg.accumulate_weights(zeros(4, 2, 40), zeros(4, 3, 4, 16), zeros(20, 8, 2, 16), zeros(4, 3, 4), table(device=device)) is None
        t, weights = bg.evict_tokens([zeros(20, 8, 2, 4)], [zeros(4, 2, 40)], table(device=device), 7)
        assert t.pages.shape == (4, 5) and [w.shape for w in weights] == [(4, 2, 40)]

    calls(lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=META), META)
    with torch._subclasses.FakeTensorMode():
        calls(lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype), "cpu")


def test_tangents():
    """Carried by rotary, refused by the others."""
    with forward_ad.dual_level():
        def dual(*s):
            return forward_ad.make_dual(torch.zeros(*s, device=META), torch.zeros(*s, device=META))

        zeros = torch.zeros(4, 2, 40, device=META)
        out, = bg.rotary([dual(2, 3, 4, 8)], torch.zeros(2, 3, dtype=I64, device=META), torch.ones(4, device=META))
        assert forward_ad.unpack_dual(out).tangent.shape == (2, 3, 4, 8)
        for call in (lambda: bg.token_logprobs(dual(4, 9), torch.zeros(4, dtype=I64, device=META)),
                     lambda: bg.rotary([dual(2, 3, 4, 8)], torch.zeros(2, 3, dtype=I64, device=META), torch.ones(4, device=META), inplace=True),
                     lambda: bg.accumulate_weights(zeros, dual(4, 3, 4, 16), torch.zeros(20, 8, 2, 16, device=META), torch.zeros(4, 3, 4, device=META),
                                                   table(device=META)),
                     lambda: bg.evict_tokens([dual(20, 8, 2, 4)], [zeros], table(device=META), 3)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()


def test_a_training_step_is_traced():
    """Forward and backward as graphs of the operators."""
    from functorch.compile import aot_function, nop

    graphs = []

    def keep(graph, _inputs):
        graphs.append({node.target for node in graph.graph.nodes})
        return nop(graph, _inputs)

    def step(x, logits, tokens, f):
        return bg.rotary([x * 2], tokens, f)[0], bg.token_logprobs(logits * 2, tokens).logprobs

    leaf, logits = (torch.zeros(*s, device=META, requires_grad=True) for s in ((2, 3, 4, 8), (2, 3, 50)))
    out = aot_function(step, fw_compiler=keep, bw_compiler=keep)(leaf, logits, torch.zeros(2, 3, dtype=I64, device=META), torch.ones(4, device=META))
    (out[0].sum() + out[1].sum()).backward()
    assert leaf.grad.shape == (2, 3, 4, 8) and logits.grad.shape == (2, 3, 50)
    ops = torch.ops.beamgrad
    assert {ops.rotary.default, ops.token_logprobs.default} <= graphs[0]
    assert {ops.rotary.default, ops.token_logprobs_backward.default} <= graphs[1]


PROBE = r"""
#include <stdio.h>
#include <string.h>
#include "beamgrad_score.h"
#include "beamgrad_state.h"
#define BAD DBS_CUDA_STATUS_INVALID_ARGUMENT
#define CHECK(x) do { if (!(x)) { printf("%s\n", #x); return 1; } } while (0)
static char room[1 << 16] __attribute__((aligned(16)));
int main(void) {
    /* scores */
    BeamgradTokenLogprobs a; memset(&a, 0, sizeof a);
    a.logits = room; a.tokens = room; a.logprobs = (float*)room; a.data_type = 2; a.outer = 3; a.inner = 5; a.vocab = 100000; a.strides[0] = 500000; a.strides[1] = 100000;
    CHECK(beamgrad_token_logprobs_workspace_size(&a) > 0);
    CHECK(beamgrad_token_logprobs(&a, 0, 0, 0) == BAD);             /* no workspace */
    CHECK(beamgrad_token_logprobs(&a, room + 1, 1 << 30, 0) == BAD); /* not aligned */
    a.top = 65; CHECK(beamgrad_token_logprobs_workspace_size(&a) == -1);
    a.top = 5; CHECK(beamgrad_token_logprobs(&a, room, 1 << 30, 0) == BAD); /* no place for the alternatives */
    a.top = 0; a.data_type = 7; CHECK(beamgrad_token_logprobs_workspace_size(&a) == -1);
    a.data_type = 2; a.outer = 1 << 20; a.inner = 16; CHECK(beamgrad_token_logprobs_workspace_size(&a) == -1);
    a.outer = 1; a.strides[0] = -1; CHECK(beamgrad_token_logprobs_workspace_size(&a) == -1);
    a.strides[0] = 0; CHECK(beamgrad_token_logprobs_backward(&a, 0, 0, 0, room, 0) == BAD); /* no stats */
    a.inner = 1; a.vocab = 1000; a.stats = (float*)(room + 8192); a.tokens = room + 8448;
    CHECK(beamgrad_token_logprobs_backward(&a, 0, 0, 0, room, 0) == BAD); /* the gradient in the logits' place */
    CHECK(beamgrad_token_logprobs_backward(&a, 0, 0, 0, room + 1998, 0) == BAD);
    /* rotary */
    const void* from[2] = {room, room + 4096}; void* to[2] = {room + 8192, room + 16384};
    int32_t heads[2] = {2, 1}, dims[2] = {16, 16}; int64_t st[6] = {96, 32, 16, 48, 16, 16}; double f[8];
    BeamgradRotary r; memset(&r, 0, sizeof r);
    r.from = from; r.to = to; r.heads = heads; r.head_dim = dims; r.from_strides = st; r.to_strides = st; r.n = 2; r.sequences = 2; r.tokens = 3;
    r.pairs = 9; r.positions = room; r.frequencies = f; r.scale = 1.0f;
    CHECK(beamgrad_rotary(&r, 0) == BAD); /* more pairs than a head has */
    r.pairs = 8; r.data_type = 9; CHECK(beamgrad_rotary(&r, 0) == BAD);
    r.data_type = 0; to[1] = room + 8192 + 64; CHECK(beamgrad_rotary(&r, 0) == BAD); /* outputs meet */
    to[1] = room + 64; CHECK(beamgrad_rotary(&r, 0) == BAD);                          /* an output in an input */
    to[0] = room; to[1] = room + 16384; CHECK(beamgrad_rotary(&r, 0) == BAD);         /* one in place, one not */
    to[1] = room + 4096; from[1] = to[1]; st[0] = 95; CHECK(beamgrad_rotary(&r, 0) == BAD); /* sequences that meet */
    st[0] = 96; r.tokens = 1 << 26; CHECK(beamgrad_rotary(&r, 0) == BAD);
    /* weights */
    BeamgradWeights w; memset(&w, 0, sizeof w);
    static char far[1 << 25] __attribute__((aligned(16))); /* keys, queries, log-sums, weights */
    w.k = far; w.q = far + (1 << 20); w.lse = (float*)(far + (1 << 22)); w.weights = (float*)(far + (1 << 23)); w.pages = w.lengths = (int32_t*)room; w.data_type = 1; w.sequences = 2; w.tokens = 600;
    w.heads = 4; w.kv_heads = 2; w.head_dim = 64; w.page_tokens = 16; w.n_pages = 100; w.table_pages = 40; w.scale = 0.125f;
    w.q_strides[0] = 153600; w.q_strides[1] = 256; w.q_strides[2] = 64; w.k_strides[0] = 2048; w.k_strides[1] = 128; w.k_strides[2] = 64;
    w.weight_strides[0] = 1280; w.weight_strides[1] = 640;
    CHECK(beamgrad_accumulate_weights_workspace_size(&w) > 0); /* many rows over few keys */
    CHECK(beamgrad_accumulate_weights_workspace_size(&w) <= 16 << 20);
    CHECK(beamgrad_accumulate_weights(&w, 0, 0, 0) == BAD);
    const int64_t bytes = beamgrad_accumulate_weights_workspace_size(&w);
    for (int i = 0; i < 3; ++i) { /* weights in keys, queries, log-sums */
        w.weights = (float*)(far + (i == 0 ? 400000 : i == 1 ? (1 << 20) + 500000 : (1 << 22) - 256));
        CHECK(beamgrad_accumulate_weights(&w, far + (1 << 24), bytes, 0) == BAD);
    }
    w.parents = (int32_t*)room; CHECK(beamgrad_accumulate_weights_workspace_size(&w) == -1); /* a tree of 600 */
    w.parents = 0; w.weight_strides[1] = 639; CHECK(beamgrad_accumulate_weights_workspace_size(&w) == -1);
    w.weight_strides[0] = 640; w.weight_strides[1] = 1280; CHECK(beamgrad_accumulate_weights_workspace_size(&w) > 0);
    w.weight_strides[1] = 640; CHECK(beamgrad_accumulate_weights_workspace_size(&w) == -1);
    w.weight_strides[1] = 1280; w.q_strides[1] = 257; CHECK(beamgrad_accumulate_weights_workspace_size(&w) == -1);
    w.q_strides[1] = 256; w.scale = -1.0f; CHECK(beamgrad_accumulate_weights_workspace_size(&w) == -1);
    w.scale = 3e38f; CHECK(beamgrad_accumulate_weights_workspace_size(&w) == -1);
    /* a long cache of many heads: no splits, no workspace */
    w.scale = 1.0f; w.table_pages = 8000; w.weight_strides[0] = 256000; w.weight_strides[1] = 128000; w.tokens = 1;
    CHECK(beamgrad_accumulate_weights_workspace_size(&w) == 0);
    /* eviction */
    void* base[2] = {room, room + 4096}; int64_t rows[2] = {32, 32}, page_stride[2] = {256, 256}, token_stride[2] = {32, 32};
    BeamgradPools p; memset(&p, 0, sizeof p);
    p.base = base; p.row_bytes = rows; p.page_stride = page_stride; p.token_stride = token_stride; p.n = 2; p.n_pages = 10; p.page_tokens = 8;
    const float* ws[2] = {(float*)(room + 8192), (float*)(room + 10000)}; float* tw[2] = {(float*)(room + 12288), (float*)(room + 16384)}; int64_t strides[4] = {80, 40, 80, 40};
    BeamgradEviction e; memset(&e, 0, sizeof e);
    e.weights = ws; e.weight_strides = strides; e.to_weights = tw; e.n_weights = 1; e.heads = 2; e.budget = 7;
    int32_t* t = (int32_t*)(room + 32768);
    BeamgradTable old = {t, t + 100, t + 200}, new = {t + 300, t + 400, t + 500};
    CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 3, 5) == 4 * (3 + 3 * 2 * 7));
    e.budgets = (int32_t*)room; CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 3, 5) == 4 * (3 + 3 * 2 * 40)); e.budgets = 0;
    CHECK(beamgrad_evict_tokens(&p, &e, &old, 3, 5, &new, 0, 0, 0) == BAD);
    CHECK(beamgrad_evict_tokens(&p, &e, &old, 3, 5, &old, room + 50000, 10000, 0) == BAD); /* the table in its own place */
    tw[0] = (float*)(room + 8192); CHECK(beamgrad_evict_tokens(&p, &e, &old, 3, 5, &new, room + 50000, 10000, 0) == BAD); /* the weights too */
    tw[0] = (float*)(room + 4096); CHECK(beamgrad_evict_tokens(&p, &e, &old, 3, 5, &new, room + 50000, 10000, 0) == BAD); /* in a pool */
    tw[0] = (float*)(room + 12288); base[1] = room + 128; CHECK(beamgrad_evict_tokens(&p, &e, &old, 3, 5, &new, room + 50000, 10000, 0) == BAD);
    base[1] = room + 4096; e.heads = 3; CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 3, 5) == -1); /* a row of no three parts */
    e.heads = 2; e.n_weights = 0; CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 3, 5) == -1);
    e.n_weights = 3; CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 3, 5) == -1);
    e.n_weights = 1; CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 65536, 5) == -1);
    e.recent = -1; CHECK(beamgrad_evict_tokens_workspace_size(&p, &e, 3, 5) == -1);
    return 0;
}
"""


def test_c_entries_refuse_before_a_launch(tmp_path):
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(PROBE)
    lib = os.path.dirname(_build.lib_path())
    subprocess.run(["gcc", "-std=gnu99", "-Wall", "-Werror", f"-I{ROOT}/include", str(src), f"-L{lib}", "-ldbs_hip",
                    f"-Wl,-rpath,{lib}", f"-L{_build.ROCM}/lib", f"-Wl,-rpath,{_build.ROCM}/lib", "-lamdhip64", "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=20)
    assert done.returncode == 0, done.stdout
