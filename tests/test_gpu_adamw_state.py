"""The optimizer's state as a mapping: complete, and without writes that are lost."""
import collections

import pytest
import torch

pytestmark = pytest.mark.gpu

NAMES = {32: ["step", "exp_avg", "exp_avg_sq"],
         8: ["step", "exp_avg", "exp_avg_sqrt", "exp_avg_scale", "exp_avg_sqrt_scale"]}


def _make(bits, step=True):
    from rexsc_b200 import optim

    g = torch.Generator(device="cuda").manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")) for s in ((300,), (17, 5), (0,), ())]
    opt = optim.AdamW([{"params": ps[:2]}, {"params": ps[2:]}], state_bits=bits)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g, device="cuda")
    if step:
        opt.step()
    return opt, ps


@pytest.mark.parametrize("bits", [32, 8])
def test_all_parameters_are_in_it(ops, bits):
    for step in (True, False):
        opt, ps = _make(bits, step)
        other = torch.nn.Parameter(torch.zeros(3, device="cuda"))
        assert all(p in opt.state for p in ps) and other not in opt.state and other.data not in opt.state
        assert len(opt.state) == 4 and bool(opt.state)
        assert [id(p) for p in opt.state] == [id(p) for p in ps] == [id(p) for p in dict(opt.state)]
        assert all(list(v) == NAMES[bits] for v in opt.state.values())
        assert opt.state.get(other) is None and opt.state.get(ps[0]) is opt.state[ps[0]]
        with pytest.raises(KeyError):
            opt.state[other]
        for p, v in opt.state.items():
            assert v["exp_avg"].shape == p.shape
        opt.add_param_group({"params": [other]})
        assert other in opt.state and len(opt.state) == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_assigned_values_are_copied(ops, bits):
    a, ps = _make(bits)
    b, qs = _make(bits, step=False)
    for q, p in zip(qs, ps):
        q.data.copy_(p.detach())
        if q is qs[0]:                                  # one by one, one after another, all at once
            for name, t in a.state[p].items():
                b.state[q][name] = t
        elif q is qs[1]:
            b.state[q].update({k: t.clone() for k, t in a.state[p].items()})
        else:
            b.state[q] = {k: t.cpu() for k, t in a.state[p].items()}
    for x, y in ((a.flat_state(i), b.flat_state(i)) for i in (0, 1)):
        for name in x:
            assert torch.equal(x[name].view(torch.uint8) if x[name].dim() else x[name], y[name].view(torch.uint8) if y[name].dim() else y[name])
    for p, q in zip(ps, qs):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    a.step()
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    b.state[qs[0]]["step"] = 10
    assert int(b.flat_state(0)["step"]) == 10
    # moving a state to the device that it is on
    for p in b.state:
        b.state[p] = {k: t.to("cuda") for k, t in b.state[p].items()}


@pytest.mark.parametrize("bits", [32, 8])
def test_refused(ops, bits):
    opt, ps = _make(bits)
    before = [t.clone() for t in opt.flat_state().values()]
    with pytest.raises(TypeError):
        opt.state = collections.defaultdict(dict)
    for change in (lambda: opt.state.clear(), lambda: opt.state.pop(ps[0]), lambda: opt.state.__delitem__(ps[0])):
        with pytest.raises((TypeError, AttributeError)):
            change()
    v = opt.state[ps[0]]
    for change in (v.clear, lambda: v.pop("step"), v.popitem, lambda: v.__delitem__("step"), lambda: v.setdefault("max", 1)):
        with pytest.raises(TypeError):
            change()
    with pytest.raises(KeyError):
        v["max_exp_avg_sq"] = torch.zeros(300, device="cuda")
    with pytest.raises(ValueError):
        v["exp_avg"] = torch.zeros(299, device="cuda")
    with pytest.raises(KeyError):
        opt.state[torch.nn.Parameter(torch.zeros(3, device="cuda"))] = {}
    for x, y in zip(before, opt.flat_state().values()):
        assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_states_hold_plain_dictionaries(ops, bits, tmp_path):
    opt, ps = _make(bits)
    sd = opt.state_dict()
    assert [type(v) for v in sd["state"].values()] == [dict] * 4
    assert all(sd["state"][0][k].data_ptr() == t.data_ptr() for k, t in opt.state[ps[0]].items())
    torch.save(sd, tmp_path / "s.pt")
    b, _ = _make(bits, step=False)
    b.load_state_dict(torch.load(tmp_path / "s.pt", weights_only=True))
    for x, y in zip(opt.flat_state().values(), b.flat_state().values()):
        assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_are_dictionaries_of_their_own(ops, bits):
    import copy
    import io

    opt, ps = _make(bits)
    views = opt.state[ps[0]]
    # (torch.save: plain pickle does not take torch's 8-bit floats)
    file = io.BytesIO()
    torch.save(views, file)
    file.seek(0)
    for other in (copy.deepcopy(views), torch.load(file, weights_only=True)):
        assert type(other) is collections.OrderedDict and list(other) == NAMES[bits]
        for name, t in other.items():
            assert t.data_ptr() != views[name].data_ptr()
            assert torch.equal(t.view(torch.uint8) if t.dim() else t, views[name].view(torch.uint8) if t.dim() else views[name])
            t.zero_()
    assert type(copy.copy(views)) is collections.OrderedDict and copy.copy(views)["step"] is views["step"]
    whole = copy.deepcopy(opt.state)
    assert type(whole) is collections.OrderedDict and len(whole) == 4
    assert all(type(v) is collections.OrderedDict for v in whole.values())
    assert int(views["step"]) == 1 and views["exp_avg"].float().abs().sum() > 0
