# SPDX-License-Identifier: MIT
"""Forward-mode derivatives and function transforms of the operators of a
model's state, by their shape-only forms: a tangent is carried or the call is
refused, never dropped."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import beamgrad_amd as bg

META = torch.device("meta")


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device=META)


def dual(*shape):
    return forward_ad.make_dual(zeros(*shape), zeros(*shape))


def calls(float_tensor):
    """Every operator without a derivative, with one tensor made by ``float_tensor``."""
    table = bg.PageTable.empty(4, 5, 20, device=META)
    ones = zeros(4, dtype=torch.int32)
    q, pool, cache, state = (zeros(*s) for s in ((4, 3, 4, 16), (20, 8, 4), (20, 8, 2, 16), (2, 3, 5)))
    parents = zeros(2, 3, dtype=torch.int64)
    return {
        "tree_attention q": lambda: bg.tree_attention(float_tensor(*q.shape), cache, cache, table),
        "tree_attention v": lambda: bg.tree_attention(q, cache, float_tensor(*cache.shape), table),
        "fork_pages": lambda: bg.fork_pages([pool, float_tensor(*pool.shape)], table, ones),
        "write_tokens pools": lambda: bg.write_tokens([float_tensor(*pool.shape)], [zeros(4, 2, 4)], table),
        "write_tokens news": lambda: bg.write_tokens([pool], [float_tensor(4, 2, 4)], table),
        "keep_tokens": lambda: bg.keep_tokens([float_tensor(*pool.shape)], table, ones, zeros(4, 2, dtype=torch.int32), ones),
        "reorder_states inplace": lambda: bg.reorder_states([state, float_tensor(*state.shape)], parents, inplace=True),
    }


NAMES = list(calls(zeros))


@pytest.mark.parametrize("gradients", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_duals_are_refused(name, gradients):
    with forward_ad.dual_level(), torch.set_grad_enabled(gradients):
        calls(zeros)[name]()
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            calls(dual)[name]()


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(name):
    """torch.func wraps its tensors: what they need is seen all the same."""
    def over(shape, transform):
        def one(x):
            calls(lambda *s: x if s == shape else zeros(*s))[name]()
            return x.sum()
        return transform(one)

    shapes = []
    calls(lambda *s: shapes.append(s) or zeros(*s))[name]()
    x = zeros(*shapes[0])
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        over(shapes[0], lambda f: torch.func.jvp(f, (x,), (x,)))
    with pytest.raises(RuntimeError, match="no gradient"):
        over(shapes[0], lambda f: torch.func.grad(f)(x))


@pytest.mark.parametrize("requires_grad", [False, True])
def test_reordered_states_carry_tangents(requires_grad):
    parents = zeros(2, 3, dtype=torch.int64)
    plain, ints = zeros(2, 3, 7), zeros(2, 3, 2, dtype=torch.int32)
    with forward_ad.dual_level():
        primal = zeros(2, 3, 5).requires_grad_(requires_grad)
        outs = bg.reorder_states([plain, forward_ad.make_dual(primal, zeros(2, 3, 5)), ints], parents)
        tangents = [forward_ad.unpack_dual(t).tangent for t in outs]
        assert tangents[0] is None and tangents[2] is None and tangents[1].shape == (2, 3, 5)
        assert outs[1].requires_grad == requires_grad and not outs[0].requires_grad
    value, tangent = torch.func.jvp(lambda x: bg.reorder_states([x], parents)[0], (plain,), (plain,))
    assert value.shape == tangent.shape == (2, 3, 7)


def test_tangents_on_the_cpu_are_refused():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(2, 3, 5), torch.zeros(2, 3, 5))
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            bg.reorder_states([x], torch.zeros(2, 3, dtype=torch.int64))


def training_step(states, parents):
    outs = bg.reorder_states([states[0] * 2, states[1]], parents)
    return torch.autograd.grad(sum((t * t).sum() for t in outs), states)


def test_the_backward_has_shapes_without_a_gpu():
    """Meta and fake tensors."""
    parents = zeros(2, 3, dtype=torch.int64)
    states = [zeros(2, 3, 5).requires_grad_(), zeros(2, 3).requires_grad_()]
    assert [g.shape for g in training_step(states, parents)] == [(2, 3, 5), (2, 3)]
    with torch._subclasses.FakeTensorMode():
        states = [torch.zeros(2, 3, 5, requires_grad=True), torch.zeros(2, 3, requires_grad=True)]
        grads = training_step(states, torch.zeros(2, 3, dtype=torch.int64))
        assert [g.shape for g in grads] == [(2, 3, 5), (2, 3)]


def test_a_training_step_is_traced():
    """Forward and backward as one graph of the two operators."""
    from functorch.compile import aot_function, nop

    graphs = []

    def keep(graph, _inputs):
        graphs.append({node.target for node in graph.graph.nodes})
        return nop(graph, _inputs)

    step = aot_function(lambda s, parents: bg.reorder_states([s * 2], parents)[0], fw_compiler=keep, bw_compiler=keep)
    leaf = zeros(2, 3, 5).requires_grad_()
    step(leaf, zeros(2, 3, dtype=torch.int64)).sum().backward()
    assert leaf.grad.shape == (2, 3, 5)
    assert torch.ops.beamgrad.reorder_states.default in graphs[0]
    assert torch.ops.beamgrad.reorder_states_backward.default in graphs[1]
