"""A weight in another order than its gradient: the same step as with the gradient in the weight's own order, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _weights(dtype):
    return [_rand((16, 8, 3, 3), 1, dtype).contiguous(memory_format=torch.channels_last), _rand((20, 30, 5), 2, dtype).permute(2, 0, 1),
            _rand((70, 33), 3, dtype).t(), _rand((999,), 4, dtype)[3:], _rand((40, 1, 7), 5, dtype), _rand((11, 13, 17, 2), 6, dtype)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype, gtype", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_order_of_the_gradient(ops, dtype, gtype, bits):
    from rexsc_b200 import optim

    start = [torch.empty_strided(w.shape, w.stride(), dtype=dtype, device="cuda").copy_(w) for w in _weights(dtype)]
    a, b, c = ([torch.nn.Parameter(torch.empty_strided(w.shape, w.stride(), dtype=dtype, device="cuda").copy_(w)) for w in start]
               for _ in range(3))
    made = [optim.AdamW(ps, lr=1e-2, state_bits=bits) for ps in (a, b, c)]
    for step in range(3):
        for i in range(len(start)):
            g = _rand(start[i].shape, 100 * step + i, gtype)
            for ps in (a, b, c):
                ps[i].grad_dtype = None
            a[i].grad = g                                                            # contiguous
            b[i].grad = torch.empty_strided(g.shape, start[i].stride(), dtype=gtype, device="cuda").copy_(g)
            assert b[i].grad.stride() == start[i].stride()
            c[i].grad = g.transpose(0, -1).contiguous().transpose(0, -1)             # in a third order
        for opt in made:
            opt.step()
    for i, w in enumerate(start):
        assert a[i].stride() == w.stride() and not torch.equal(a[i].detach(), w)
        assert torch.equal(a[i], b[i]) and torch.equal(a[i], c[i])
    for other in made[1:]:
        for x, y in zip(made[0].flat_state().values(), other.flat_state().values()):
            assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)
    # and the update of the same values in a contiguous weight (32 bits: each element by itself)
    if bits == 32:
        plain = [torch.nn.Parameter(w.contiguous().clone()) for w in start]
        opt = optim.AdamW(plain, lr=1e-2, state_bits=32)
        for step in range(3):
            for i, p in enumerate(plain):
                p.grad_dtype = None
                p.grad = _rand(start[i].shape, 100 * step + i, gtype)
            opt.step()
        assert all(torch.equal(p, q) for p, q in zip(a, plain))
