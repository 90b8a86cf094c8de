"""Very small eps: weights whose gradient has always been 0 stay finite, as 0 / eps is 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-37, 1e-30, 1e-8])
def test_gradients_of_0(ops, bits, eps):
    from rexsc_b200 import optim

    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    opt = optim.AdamW([p], lr=0.1, weight_decay=0.0, eps=eps, state_bits=bits)
    for _ in range(3):
        p.grad = torch.zeros_like(p)
        p.grad[::7] = 1.0
        opt.step()
    changed = torch.zeros(1000, dtype=torch.bool, device="cuda")
    changed[::7] = True
    assert (p[~changed] == 1).all() and p.isfinite().all() and (p[changed] < 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_refused(ops, bits):
    from rexsc_b200 import optim

    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    for eps in (1e-40, 1e-50):
        with pytest.raises(ValueError):
            optim.AdamW([p], eps=eps, state_bits=bits)
    opt = optim.AdamW([p], state_bits=bits)
    opt.param_groups[0]["eps"] = 1e-40                    # found by the step
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError):
        opt.step()
    assert (p == 1).all()
