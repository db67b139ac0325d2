# SPDX-License-Identifier: MIT
"""Which captured backwards of reordered states are refused: those that reach a
leaf that a living graph of another stream holds, through any operators. Outside a
capture, where the question is the same."""

import pytest
import torch

import beamgrad_amd as bg

pytestmark = pytest.mark.gpu

PARENTS = [[0, 0, 2, 1]]
ROUTES = {
    "direct": lambda leaf: bg.reorder_states([leaf], torch.tensor(PARENTS).cuda())[0],
    "expanded": lambda leaf: bg.reorder_states([leaf[:, :1].expand(1, 4, 8)], torch.tensor(PARENTS).cuda())[0],
    "scaled": lambda leaf: bg.reorder_states([torch.ones(1, 4, 8, device="cuda"), leaf * 3.0], torch.tensor(PARENTS).cuda())[1],
    "cast": lambda leaf: bg.reorder_states([leaf.bfloat16()], torch.tensor(PARENTS).cuda())[0].float().sum(),
    "twice": lambda leaf: ROUTES["scaled"](ROUTES["direct"](leaf)),
}


@pytest.mark.parametrize("route", list(ROUTES))
def test_a_leaf_is_found_through_other_operators(route):
    leaf = torch.randn(1, 4, 8, device="cuda").requires_grad_()
    free = torch.randn(1, 4, 8, device="cuda").requires_grad_()
    alive = ROUTES[route](leaf)
    reaches = torch.ops.beamgrad.backward_reaches_leaf_of_another_stream
    assert not reaches(alive)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = ROUTES[route](leaf)
        assert reaches(out)
        assert not reaches(ROUTES[route](free))
        assert reaches(ROUTES[route](free) + out)
        assert not reaches(free) and not reaches(out.detach())
        del out, alive
        assert not reaches(ROUTES[route](leaf))
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()


def test_a_backward_through_other_operators_is_captured():
    """A leaf behind another operator, held by no other graph."""
    parents = torch.tensor(PARENTS).cuda()
    x = torch.randn(1, 4, 8, device="cuda").requires_grad_()
    g = torch.randn(1, 4, 8, device="cuda")

    def step():
        out = bg.reorder_states([x * 2], parents)[0]
        return torch.autograd.grad(out, x, g)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step()
    for seed in range(3):
        g.copy_(torch.randn(1, 4, 8, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, step())
