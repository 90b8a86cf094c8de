"""Weights that come to share memory after the optimizer was made, and gradients that lie in weights' memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _rand(n, dtype=F32, seed=0):
    return torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _make(params, bits):
    from rexsc_b200 import optim

    return optim.AdamW(params, lr=0.1, state_bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_weights_given_the_same_memory(ops, bits):
    ps = [torch.nn.Parameter(_rand(700, seed=i)) for i in range(4)]
    opt = _make(ps, bits)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    before = [p.detach().clone() for p in ps]
    own = ps[2].data
    flat = _rand(1400, seed=9)
    for tied in (ps[0].data, flat[500:1200]):
        ps[2].data = tied
        ps[1].data = flat[:700] if tied is not ps[0].data else before[1].clone()
        now = [p.detach().clone() for p in ps]
        versions = [p._version for p in ps]
        with pytest.raises(ValueError, match="share memory"):
            opt.step()
        assert all(torch.equal(p.detach(), n) for p, n in zip(ps, now)) and [p._version for p in ps] == versions
    ps[2].grad, ps[1].grad = None, None                # neither is written to: nothing is shared
    opt.step()
    ps[2].data, ps[1].data = own, flat[:700]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()                                         # other memory, in another order, is fine
    ps[0].data, ps[3].data = ps[3].data, ps[0].data
    opt.step()
    assert int(opt.flat_state()["step"]) == 4


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_in_weights_memory(ops, bits, dtype):
    """The step of gradients that have memory of their own.  Large enough that some blocks are written long before others read."""
    n = 3_000_000

    def step(alias):
        a, b, c = (torch.nn.Parameter(_rand(n, dtype, i)) for i in range(3))
        store = torch.zeros(n + 64, device="cuda", dtype=dtype)
        d = torch.nn.Parameter(store[:n].copy_(_rand(n, dtype, 3)))
        opt = _make([a, b, c, d], bits)
        own = (lambda t: t) if alias else torch.clone
        a.grad, b.grad = own(c.detach()), own(a.detach())
        c.grad = own(c.detach())                       # its own memory
        d.grad = own(store[64:])                       # its own memory, shifted
        opt.step()
        return [t.detach().clone() for t in (a, b, c, d)] + [t.view(torch.uint8).clone() if t.dim() else t.clone() for t in opt.flat_state().values()]

    for x, y in zip(step(True), step(False)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_share_memory_with_one_another(ops, bits):
    """Only read: views of one buffer, and the same tensor for two weights."""
    def step(alias):
        ps = [torch.nn.Parameter(_rand(700, seed=i)) for i in range(3)]
        opt = _make(ps, bits)
        flat = _rand(1400, seed=5)
        for p, g in zip(ps, (flat[:700], flat[350:1050], flat[:700])):
            p.grad = g if alias else g.clone()
        opt.step()
        return [p.detach().clone() for p in ps]

    for x, y in zip(step(True), step(False)):
        assert torch.equal(x, y)
