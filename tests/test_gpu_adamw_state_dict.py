"""Hooks of state_dict(): they see all of it, and may return another one."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _make(bits=32):
    from rexsc_b200 import optim

    ps = [torch.nn.Parameter(torch.ones(s, device="cuda")) for s in ((300,), (7, 5), (4,))]
    opt = optim.AdamW([{"params": ps[:1]}, {"params": ps[1:], "lr": 0.5}], lr=0.25, state_bits=bits)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    return opt, ps


@pytest.mark.parametrize("bits", [32, 8])
def test_post_hooks_see_all_of_it(ops, bits):
    opt, _ = _make(bits)
    plain = opt.state_dict()
    seen = []
    opt.register_state_dict_pre_hook(lambda o: seen.append("pre"))
    opt.register_state_dict_post_hook(lambda o, sd: seen.append(copy.deepcopy(sd)))
    sd = opt.state_dict()
    assert seen[0] == "pre" and len(seen) == 2
    other, _ = _make(bits)
    for got in (sd, seen[1]):
        assert list(got) == list(plain) and got["param_groups"] == plain["param_groups"] and list(got["state"]) == [0, 1, 2]
        for t in other.flat_state().values():
            t.zero_()
        other.load_state_dict(got)                 # what a hook has taken can be loaded
        for x, y in zip(opt.flat_state().values(), other.flat_state().values()):
            assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)


def test_post_hooks_may_return_another_state(ops):
    opt, _ = _make()
    opt.register_state_dict_post_hook(lambda o, sd: {"inner": sd})
    opt.register_state_dict_post_hook(lambda o, sd: {"outer": sd})
    assert opt.state_dict()["outer"]["inner"]["state_bits"] == 32


def test_the_same_entries_as_torchs(ops):
    opt, ps = _make()
    ref = torch.optim.AdamW([{"params": ps[:1]}, {"params": ps[1:], "lr": 0.5}], lr=0.25)
    ref.step()
    mine, theirs = opt.state_dict(), ref.state_dict()
    assert set(theirs) <= set(mine) and list(mine["state"]) == list(theirs["state"])
    for a, b in zip(mine["param_groups"], theirs["param_groups"]):
        assert a["params"] == b["params"] and a["lr"] == b["lr"] and a["betas"] == b["betas"]
    for a, b in zip(mine["state"].values(), theirs["state"].values()):
        assert set(a) == set(b) and all(a[k].shape == b[k].shape for k in a)
    # a dictionary of its own: changes do not reach the optimizer
    mine["param_groups"][0]["lr"] = 9.0
    mine["param_groups"][0]["params"].append(7)
    mine["state"].clear()
    assert opt.param_groups[0]["lr"] == 0.25 and len(opt.param_groups[0]["params"]) == 1 and len(opt.state) == 3
