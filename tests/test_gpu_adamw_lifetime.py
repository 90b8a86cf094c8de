"""An optimizer's memory is given back when it is dropped, without a garbage collection."""
import gc
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("used", [False, True])
def test_dropped_optimizers(ops, bits, used):
    from rexsc_b200 import optim

    p = torch.nn.Parameter(torch.zeros(4 << 20, device="cuda"))
    p.grad = torch.ones_like(p)
    # (the first optimizer of a process, of whatever kind, stays in frames of an import that torch then does)
    torch.optim.SGD([p], lr=0.1)
    gc.collect()
    gc.disable()
    try:
        before = torch.cuda.memory_allocated()
        opt = optim.AdamW([p], state_bits=bits)
        opt.step()
        if used:
            assert opt.state[p]["exp_avg"].shape == p.shape
            opt.load_state_dict(opt.state_dict())
        held = torch.cuda.memory_allocated() - before
        assert held >= (4 << 20) * (8 if bits == 32 else 2)
        gone = weakref.ref(opt)
        del opt
        assert gone() is None
        assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()


@pytest.mark.parametrize("bits", [32, 8])
def test_views_outlive_it(ops, bits):
    from rexsc_b200 import optim

    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p], state_bits=bits)
    opt.step()
    state, m = opt.state, opt.state[p]["exp_avg"]
    copy = m.float().clone()
    del opt
    torch.zeros(10000, device="cuda")
    assert torch.equal(m.float(), copy) and torch.equal(state[p]["exp_avg"].float(), copy) and int(state[p]["step"]) == 1
