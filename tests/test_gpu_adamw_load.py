"""What loading a state takes over: values, and none of the checkpoint's tensors; hooks as torch's optimizers call them."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _make(lr, bits=32, seed=0, **kw):
    from rexsc_b200 import optim

    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(700, generator=g, device="cuda"))
    p.grad = torch.randn(700, generator=g, device="cuda")
    return optim.AdamW([p], lr=lr, state_bits=bits, **kw), p


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_reads_the_loaded_lr(ops, bits):
    saved, _ = _make(torch.tensor(0.25, device="cuda"), bits)
    saved.step()
    lr = torch.tensor(1e-3, device="cuda")
    opt, p = _make(lr, bits, seed=1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(saved.state_dict())
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.25
    ref, q = _make(0.25, bits, seed=1)
    ref.load_state_dict(copy.deepcopy({**saved.state_dict()}))
    q.data.copy_(p.detach())
    graph.replay()
    ref.step()
    assert torch.equal(p, q)
    # a number loaded over a tensor
    plain, _ = _make(0.125, bits)
    opt.load_state_dict(plain.state_dict())
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.125


@pytest.mark.parametrize("mine", [1e-3, "tensor"])
def test_nothing_of_the_checkpoint_is_shared(ops, mine):
    saved, _ = _make(torch.tensor(0.25, device="cuda"))
    saved.step()
    sd = saved.state_dict()
    opt, p = _make(torch.tensor(1e-3, device="cuda") if mine == "tensor" else mine)
    opt.load_state_dict(sd)
    sd["param_groups"][0]["lr"].fill_(9.0)                # the checkpoint's, and the saved optimizer's own
    saved.param_groups[0]["lr"].fill_(9.0)
    for t in sd["state"][0].values():
        t.zero_()
    assert float(opt.param_groups[0]["lr"]) == 0.25
    assert float(opt.flat_state()["exp_avg"].abs().sum()) > 0 and int(opt.flat_state()["step"]) == 1
    before = p.detach().clone()
    opt.step()
    assert 0.01 < float((p.detach() - before).abs().max()) < 1.0


def test_hooks(ops):
    for make in (lambda: _make(0.5)[0], lambda: torch.optim.AdamW([torch.nn.Parameter(torch.zeros(700, device="cuda"))], lr=0.5)):
        opt, other, seen = make(), make(), []

        def pre(o, sd):
            assert o is opt
            seen.append("pre")
            groups = copy.deepcopy(sd["param_groups"])
            groups[0]["lr"] = 0.75
            return {**sd, "param_groups": groups}

        def later(o, sd):
            seen.append(sd["param_groups"][0]["lr"])
            sd["param_groups"][0]["lr"] = 0.875           # (in place: of the dict that the hook before it made)

        def post(o):
            assert o is opt
            seen.append(("post", o.param_groups[0]["lr"]))

        opt.register_load_state_dict_pre_hook(pre)
        opt.register_load_state_dict_pre_hook(later)
        opt.register_load_state_dict_post_hook(post)
        sd = other.state_dict()
        opt.load_state_dict(sd)
        assert seen == ["pre", 0.75, ("post", 0.875)]
        assert sd["param_groups"][0]["lr"] == 0.5


def test_hooks_that_replace_keys_leave_the_callers_state(ops):
    opt, _ = _make(0.5)
    opt.register_load_state_dict_pre_hook(lambda o, sd: sd.pop("extra", None) and None)
    sd = {**_make(0.25)[0].state_dict(), "extra": 1}
    opt.load_state_dict(sd)
    assert sd["extra"] == 1 and opt.param_groups[0]["lr"] == 0.25


def test_names_of_parameters_stay(ops):
    from rexsc_b200 import optim

    def make(name):
        return optim.AdamW([(name, torch.nn.Parameter(torch.zeros(5, device="cuda")))])

    a, b = make("head"), make("tail")
    b.load_state_dict(a.state_dict())
    assert b.param_groups[0]["param_names"] == ["tail"]


@pytest.mark.parametrize("mine", [(), (1,), (1, 1)])
@pytest.mark.parametrize("theirs", [(), (1,), "number", "cpu"])
def test_shapes_of_a_tensor_lr(ops, mine, theirs):
    value = 0.25 if theirs == "number" else torch.tensor(0.25) if theirs == "cpu" else torch.full(theirs, 0.25, device="cuda")
    saved, _ = _make(value)
    saved.step()
    lr = torch.full(mine, 1e-3, device="cuda")
    opt, p = _make(lr)
    opt.load_state_dict(saved.state_dict())
    assert opt.param_groups[0]["lr"] is lr and lr.shape == mine and float(lr) == 0.25
    opt.step()
    assert int(opt.flat_state()["step"]) == 2
