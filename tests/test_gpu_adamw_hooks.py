"""Hooks of a step and of its closure, as torch's optimizers call them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _both():
    """torch's AdamW and this library's, over the same weight and gradient."""
    from rexsc_b200 import optim

    out = []
    for make in (torch.optim.AdamW, optim.AdamW):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 300, device="cuda"))
        p.grad = torch.ones_like(p)
        out.append((make([p], lr=0.1), p))
    return out


def _seen(opt, p, call, changes):
    """What the hooks of ``call`` are given and what it returns; ``changes``: what the pre-hook makes of the arguments."""
    seen = []

    def pre(o, args, kwargs):
        assert o is opt and args[0] is opt
        seen.append(("pre", args[1:], dict(kwargs)))
        return changes(args, kwargs)

    def post(o, args, kwargs):
        assert o is opt and args[0] is opt
        seen.append(("post", args[1:], dict(kwargs)))

    handles = [opt.register_step_pre_hook(pre), opt.register_step_post_hook(post)]
    before = p.detach().clone()
    loss = call(opt)
    for h in handles:
        h.remove()
    assert not torch.equal(p.detach(), before)
    return seen, loss


def _closure():
    return 5.0


def _other():
    return 7.0


@pytest.mark.parametrize("changes", [
    lambda args, kwargs: None, lambda args, kwargs: (args, kwargs), lambda args, kwargs: (args[:1], {}),
    lambda args, kwargs: (args[:1], {"closure": _other}), lambda args, kwargs: ((args[0], _other), {}),
    lambda args, kwargs: ((args[0], None), {}), lambda args, kwargs: (args[:1], {"closure": None})])
@pytest.mark.parametrize("call", [lambda o: o.step(), lambda o: o.step(_closure)])
def test_arguments_that_hooks_see_and_return(ops, call, changes):
    theirs, ours = (_seen(opt, p, call, changes) for opt, p in _both())
    assert ours == theirs


def test_a_closure_by_keyword(ops):
    for opt, p in _both():
        assert opt.step(closure=_closure) == 5.0


def test_hooks_that_return_something_else(ops):
    for opt, p in _both():
        for bad in (3, (1,), [(opt,), {}], ((opt, _closure, 1), {}), ((opt,), {"loss": 1})):
            handle = opt.register_step_pre_hook(lambda o, args, kwargs: bad)
            with pytest.raises((RuntimeError, TypeError)):
                opt.step()
            handle.remove()
        opt.step()


def test_hooks_of_all_optimizers(ops):
    from torch.optim.optimizer import register_optimizer_step_post_hook, register_optimizer_step_pre_hook

    results = []
    for opt, p in _both():
        seen = []
        handles = [register_optimizer_step_pre_hook(lambda o, args, kwargs: (args[:1], {"closure": _other})),
                   opt.register_step_pre_hook(lambda o, args, kwargs: seen.append(dict(kwargs))),
                   opt.register_step_post_hook(lambda o, args, kwargs: seen.append("own")),
                   register_optimizer_step_post_hook(lambda o, args, kwargs: seen.append("all"))]
        seen.append(opt.step())
        for h in handles:
            h.remove()
        results.append(seen)
    assert results[0] == results[1]
