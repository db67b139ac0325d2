# SPDX-License-Identifier: MIT
"""Forward-mode derivatives of reordered states on the GPU, against the plain
restatement."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import beamgrad_amd as bg
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

PARENTS = torch.tensor([[0, 0, -1, 1], [3, 3, 3, 7]])


def draw(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
def test_tangents_move_as_the_states_do(dtype):
    x, t, plain = draw(0, 2, 4, 7, dtype=dtype), draw(1, 2, 4, 7, dtype=dtype), draw(2, 2, 4, 3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.cuda(), t.cuda())
        outs = bg.reorder_states([plain.cuda(), dual], PARENTS.cuda())
        assert forward_ad.unpack_dual(outs[0]).tangent is None
        primal, tangent = forward_ad.unpack_dual(outs[1])
        assert torch.equal(primal.cpu(), ref.reorder(x, PARENTS)) and torch.equal(tangent.cpu(), ref.reorder(t, PARENTS))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            bg.reorder_states([dual], PARENTS.cuda(), inplace=True)
    value, tangent = torch.func.jvp(lambda s: bg.reorder_states([s * 2], PARENTS.cuda())[0], (x.cuda(),), (t.cuda(),))
    assert torch.equal(value.cpu(), ref.reorder(x * 2, PARENTS)) and torch.equal(tangent.cpu(), ref.reorder(t * 2, PARENTS))


def test_tangents_with_gradients():
    """Reverse mode of a tangent, and forward mode of a gradient."""
    x, t, w = (draw(s, 2, 4, 5).cuda() for s in range(3))
    weights = t.clone().requires_grad_()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, weights)
        tangent = forward_ad.unpack_dual(bg.reorder_states([dual], PARENTS.cuda())[0]).tangent
        (grad,) = torch.autograd.grad(tangent, weights, w)
    assert torch.allclose(grad.cpu().double(), ref.reorder_gradient(w.cpu(), PARENTS)[0], atol=1e-6)
    # the gradient of sum(y^2 w) / 2 in x is the gather of y w, whose tangent along t is that of (reorder t) w
    leaf = x.clone().requires_grad_()
    with forward_ad.dual_level():
        y = bg.reorder_states([forward_ad.make_dual(leaf, t)], PARENTS.cuda())[0]
        (grad,) = torch.autograd.grad((y * y * w).sum() / 2, leaf)
        tangent = forward_ad.unpack_dual(grad).tangent
    want = ref.reorder_gradient(ref.reorder(t.cpu(), PARENTS) * w.cpu(), PARENTS)[0]
    assert torch.allclose(tangent.cpu().double(), want, atol=1e-5)


def test_a_compiled_training_step():
    """Forward and backward traced together give what they give untraced."""
    def step(x):
        return bg.reorder_states([x * 2], PARENTS.cuda())[0]

    x, w = draw(0, 2, 4, 5).cuda(), draw(1, 2, 4, 5).cuda()
    want = x.clone().requires_grad_()
    (step(want) * w).sum().backward()
    got = x.clone().requires_grad_()
    (torch.compile(step, backend="aot_eager", fullgraph=True)(got) * w).sum().backward()
    assert torch.equal(got.grad, want.grad)
