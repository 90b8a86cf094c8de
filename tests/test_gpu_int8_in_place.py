"""Outputs of int8_linear that a program changes in place: they are tensors of their own, whatever x's shape."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(64,), (5, 64), (2, 3, 64), (2, 1, 4, 64), (0, 3, 64)]


def _rand(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("prepared", [False, True])
def test_training(ops, shape, prepared):
    x, w, b = _rand(shape, 1), _rand((40, 64), 2), _rand((40,), 3)
    dy, other = _rand((*shape[:-1], 40), 4), _rand((*shape[:-1], 40), 5)

    def grads(after):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, other)]
        y = ops.int8_linear(leaves[0], ops.int8_quantize(w) if prepared else leaves[1], leaves[2])
        assert not y._is_view()
        z = after(y, leaves[3])
        return [z.detach(), *torch.autograd.grad(z, leaves, dy, allow_unused=True)]

    for inside, outside in [(lambda y, o: y.relu_(), lambda y, o: y.relu()), (lambda y, o: y.add_(o), lambda y, o: y + o),
                            (lambda y, o: y.mul_(2).add_(o).relu_(), lambda y, o: (y * 2 + o).relu())]:
        for a, c in zip(grads(inside), grads(outside)):
            assert (a is None) == (c is None)
            assert a is None or torch.equal(a, c)


@pytest.mark.parametrize("shape", SHAPES)
def test_frozen_layers_beside_one_that_is_trained(ops, shape):
    """Nothing here requires a gradient, but grad mode is on: what is added to the output may."""
    x, w = _rand(shape, 1), _rand((40, 64), 2)
    for weight in (w, ops.int8_quantize(w)):
        y, ref = ops.int8_linear(x, weight), ops.int8_linear(x, weight)
        assert not y._is_view() and not y.requires_grad
        adapter = _rand((40,), 3).requires_grad_()
        y += adapter
        assert torch.equal(y, ref + adapter)
        y.sum().backward()
        assert torch.equal(adapter.grad, torch.full((40,), float(x.numel() // 64), device="cuda"))
        with torch.no_grad():
            z = ops.int8_linear(x, weight)
        z += adapter
        assert z.requires_grad


@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_are_tensors_of_their_own(ops, shape):
    x, w = _rand(shape, 1).requires_grad_(), _rand((40, 64), 2).requires_grad_()
    ops.int8_linear(x, w).sum().backward()
    for t in (x, w):
        assert t.grad.shape == t.shape and t.grad.is_contiguous() and not t.grad._is_view()
        factor = torch.ones((), device="cuda", requires_grad=True)
        t.grad.mul_(factor)
        assert t.grad.requires_grad
