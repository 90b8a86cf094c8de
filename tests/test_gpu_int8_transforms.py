"""Forward-mode derivatives and traces of the int8 ops: there are none, and a call says so instead of leaving them out."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def _rand(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(ops, which, grad):
    given = {"x": _rand((4, 64), 1), "weight": _rand((40, 64), 2), "bias": _rand((40,), 3)}
    ref = ops.int8_linear(**given)
    with fwd.dual_level():
        dual = dict(given)
        dual[which] = fwd.make_dual(given[which].clone().requires_grad_(grad), torch.ones_like(given[which]))
        with pytest.raises(NotImplementedError):
            ops.int8_linear(**dual)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            ops.int8_linear(**dual)
        if which != "weight":
            with pytest.raises(NotImplementedError):
                ops.int8_linear(**{**dual, "weight": ops.int8_quantize(given["weight"])})
        assert torch.equal(ops.int8_linear(**given), ref)                # others are computed as before
        plain = {k: fwd.unpack_dual(v).primal.detach() for k, v in dual.items()}
        assert torch.equal(ops.int8_linear(**plain), ref)
        with torch.inference_mode():                                     # where no tangents are kept
            assert torch.equal(ops.int8_linear(**given), ref)


def test_transforms_of_functions_raise(ops):
    x, w = _rand((4, 64), 1), _rand((40, 64), 2)
    w8 = ops.int8_quantize(w)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ops.int8_linear(t, w8), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: ops.int8_linear(t, w8))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ops.int8_linear(t, w8).sum())(x)


@pytest.mark.filterwarnings("ignore")
def test_traces_are_refused(ops):
    x, w = _rand((4, 64), 1), _rand((40, 64), 2)
    w8 = ops.int8_quantize(w)
    q, s = w8.values(), w8.scale
    for f in (lambda t: ops.int8_linear(t, w8), lambda t: ops.int8_linear(t, w), lambda t: ops.int8_quantize(t).scale,
              lambda t: t + ops.int8_matmul(w8, w8)[0, 0], lambda t: t + w8.values()[0, 0],
              lambda t: t + ops.Int8Matrix.from_values(q, s).scale[0]):
        with pytest.raises(NotImplementedError):
            torch.jit.trace(f, (x,))
    assert ops.int8_linear(x, w8).shape == (4, 40)
