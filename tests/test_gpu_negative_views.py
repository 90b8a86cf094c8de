"""Real tensors that are negative views of memory (the imaginary part of a conjugate): their values count, not the memory's."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _neg(t):
    """A view with the values of ``t`` whose memory holds -t."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_int8_ops(ops, dtype):
    x, w, b, dy = _rand((5, 64), 1, dtype), _rand((40, 64), 2, dtype), _rand((40,), 3, dtype), _rand((5, 40), 4, dtype)
    w8 = ops.int8_quantize(w)
    other = ops.int8_quantize(_neg(w))
    assert torch.equal(other.values(), w8.values()) and torch.equal(other.scale, w8.scale)
    ref = ops.int8_linear(x, w8, b)
    assert torch.equal(ops.int8_linear(_neg(x), w8, b), ref)
    assert torch.equal(ops.int8_linear(x, w8, _neg(b)), ref)
    assert torch.equal(ops.int8_linear(_neg(x), _neg(w), _neg(b)), ref)
    assert torch.equal(ops.int8_matmul(w8, w8, _neg(b)), ops.int8_matmul(w8, w8, b))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops.int8_linear(*leaves), leaves, dy)
    leaves = [_neg(t).detach().requires_grad_() for t in (x, w, b)]
    y = ops.int8_linear(*leaves)
    assert torch.equal(y.detach(), ref)
    for a, c in zip(torch.autograd.grad(y, leaves, _neg(dy)), want):
        assert torch.equal(a, c)
    z = torch.complex(_rand((7, 1), 5), _rand((7, 1), 6))
    column = z.conj().imag
    assert column.is_neg()
    assert torch.equal(ops.int8_quantize(column).values(), ops.int8_quantize(column.resolve_neg()).values())


def test_matrices(ops):
    v = torch.randint(-127, 128, (30, 50), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.int8)
    s = torch.rand(30, device="cuda")
    m = ops.Int8Matrix.from_values(torch._neg_view(-v), _neg(s))
    assert torch.equal(m.values(), v) and torch.equal(m.scale, s)
    with pytest.raises(ValueError):
        ops.Int8Matrix(30, 50, m.data, _neg(s))
    with pytest.raises(ValueError):
        ops.Int8Matrix(30, 50, torch._neg_view(m.data), m.scale)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(ops, bits):
    from rexsc_b200 import optim

    out = []
    for view in (lambda t: t, _neg):
        p, q = torch.nn.Parameter(_rand((700,), 1)), torch.nn.Parameter(_rand((9, 30), 2))
        opt = optim.AdamW([p, q], lr=view(torch.tensor(0.1, device="cuda")), state_bits=bits)
        p.grad, q.grad = view(_rand((700,), 3)), view(_rand((9, 30), 4))
        opt.grad_scale, opt.found_inf = view(torch.tensor(4.0, device="cuda")), torch.zeros((), device="cuda")
        opt.step()
        out.append((p.detach(), q.detach()))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch._neg_view(_rand((700,), 1)))], state_bits=bits)
