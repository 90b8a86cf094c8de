"""AdamW steps against their definition in 64 bits.

With u = 2^-24: a step adds at most four roundings (constants, products, sum) to each 32-bit moment, of the magnitudes that are
added up, so t steps leave m and v off by 4 t u of them.  A weight's change m / root of v is off by 4 t u + 2 t u for those and
by less than 24 u for what follows (the corrections' expm1f 2 ulp and its argument, the reciprocal root 2 ulp, the quotient 2
ulp, the constants and products); the weight itself by its product with 1 - lr wd, that constant and its own rounding, 4 u.  8-bit moments are decided by values that the operator holds in fp32 after every
operation, so a restatement with the same roundings has to give the same codes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 0.1


@pytest.fixture()
def optim(ops):
    from rexsc_b200 import optim as _optim

    return _optim


def _rand(shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _f32(x):
    return x.float().double()


class Ref:
    """One tensor's AdamW in 64 bits; ``first``: place of its first element in the flat buffers (8-bit moments)."""

    def __init__(self, p, bits, first=0):
        self.p, self.bits, self.first = p.detach().double().reshape(-1).clone(), bits, first
        self.dtype, self.t, n = p.dtype, 0, p.numel()
        self.m, self.v = torch.zeros(n, device="cuda").double(), torch.zeros(n, device="cuda").double()
        self.pad = -n % 256
        blocks = (n + self.pad) // 256
        self.m8, self.r8 = (torch.zeros(blocks, 256, device="cuda").double() for _ in range(2))
        self.ms, self.rs = (torch.zeros(blocks, 1, device="cuda").double() for _ in range(2))
        self.change = torch.zeros_like(self.p)
        self.mag = torch.zeros_like(self.p)     # magnitudes that m adds up

    def step(self, g, unscale=1.0, lr=LR, wd=WD):
        self.t += 1
        g = _f32(g.double().reshape(-1) * unscale)
        self.mag = B1 * self.mag + (1 - B1) * g.abs()
        n = g.numel()
        if self.bits == 8:
            b1, c1, b2, c2 = (float(torch.tensor(c, dtype=F32)) for c in (B1, 1 - B1, B2, 1 - B2))
            gp = torch.cat([g, g.new_zeros(self.pad)]).view(-1, 256)
            m = _f32(self.m8 * self.ms)
            v = _f32(_f32(self.r8 * self.rs) ** 2)
            m = _f32(_f32(b1 * m) + _f32(c1 * gp))
            r = _f32(_f32(_f32(b2 * v) + _f32(c2 * _f32(gp * gp))).sqrt())
            i = torch.arange(m.numel(), device="cuda").view(-1, 256) + self.first
            u = (i * 0xC13FA9A9 + self.t * 0x9E3779B9) % 2 ** 32
            self.m8, self.ms = self._store(m, u // 4096, False)
            self.r8, self.rs = self._store(r, (2 ** 32 - 1 - u) // 4096, True)
            m, r = m.view(-1)[:n], r.view(-1)[:n]
        else:
            self.m = m = B1 * self.m + (1 - B1) * g
            self.v = B2 * self.v + (1 - B2) * g * g
            r = self.v.sqrt()
        per = lr / (1 - B1 ** self.t) / (r / math.sqrt(1 - B2 ** self.t) + EPS)
        self.change = per * torch.maximum(self.mag, m.abs())
        self.p = self.p * (1 - lr * wd) - per * m

    @staticmethod
    def _store(x, u, floor):
        a = x.abs().amax(1, keepdim=True)
        live = a >= 2.0 ** -100
        a1 = torch.where(live, a, 1.0)
        y = torch.where(live, _f32(x.abs() * _f32(448 / a1)), 0.0)
        step = torch.exp2((torch.frexp(y).exponent - 4).clamp(min=-9).double())
        # (below 2^-6 the sum of the fraction and u is held in fp32; it has at most 24 bits only above 2^-3, where it may round)
        cut = torch.where(y < 2.0 ** -6, _f32(_f32(y * 512) + u.double() / 2 ** 20).floor(), (y / step + u.double() / 2 ** 20).floor())
        code = (cut * step).clamp(max=448)
        if floor:
            code = torch.where(y > 0, code.clamp(min=2.0 ** -9), code)
        return code * x.sign(), torch.where(live, _f32(a / 448), 0.0)


def _check_p(p, ref, steps=1):
    err = (p.detach().double().reshape(-1) - ref.p).abs()
    allowed = steps * ((6 * ref.t + 24) * 2.0 ** -24 * ref.change + 4 * 2.0 ** -24 * ref.p.abs()) + 1e-30
    if p.dtype != F32:
        info = torch.finfo(p.dtype)
        allowed = allowed + ref.p.abs() * info.eps * 0.5001 + info.smallest_normal * info.eps / 2
    assert (err <= allowed).all(), float((err / allowed).max())


def _make(optim, params, bits, **kw):
    return optim.AdamW(params, **{**dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits), **kw})


def _firsts(params):
    at, out = 0, []
    for p in params:
        out.append(at)
        at += -(-p.numel() // 256) * 256
    return out


def _check_state(opt, params, refs, bits, steps):
    for p, r in zip(params, refs):
        s = opt.state[p]
        n = p.numel()
        if bits == 32:
            assert ((s["exp_avg"].double().reshape(-1) - r.m).abs() <= steps * 4 * 2.0 ** -24 * r.mag).all()
            assert ((s["exp_avg_sq"].double().reshape(-1) - r.v).abs() <= steps * 4 * 2.0 ** -24 * r.v).all()
        else:
            assert torch.equal(s["exp_avg"].double().reshape(-1), r.m8.view(-1)[:n])
            assert torch.equal(s["exp_avg_sqrt"].double().reshape(-1), r.r8.view(-1)[:n])
            assert torch.equal(s["exp_avg_scale"].double(), r.ms.view(-1))
            assert torch.equal(s["exp_avg_sqrt_scale"].double(), r.rs.view(-1))
        assert int(s["step"]) == steps


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype, gtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
def test_steps_against_the_definition(optim, dtype, gtype, bits):
    sizes = [(1,), (7,), (255,), (256,), (257,), (64, 3, 7, 7), (1000,), (1000, 512), (3, 5, 11), (2, 2048)]
    params = [torch.nn.Parameter(_rand(s, dtype, i, 0.1)) for i, s in enumerate(sizes)]
    opt = _make(optim, params, bits)
    refs = [Ref(p, bits, f) for p, f in zip(params, _firsts(params))]
    for step in range(4):
        for i, (p, r) in enumerate(zip(params, refs)):
            p.grad_dtype = None
            p.grad = _rand(p.shape, gtype, 100 * step + i, 10.0 ** (i % 5 - 3))
            r.p = p.detach().double().reshape(-1)   # (16-bit weights are rounded at every step)
            r.step(p.grad)
        opt.step()
        for p, r in zip(params, refs):
            _check_p(p, r)
        _check_state(opt, params, refs, bits, step + 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_gaps(optim, bits):
    # more tensors than a launch takes, some without a gradient: their moments and weights stay
    params = [torch.nn.Parameter(_rand((1 + (i * 37) % 700,), F32, i)) for i in range(1500)]
    opt = _make(optim, params, bits)
    refs = [Ref(p, bits, f) for p, f in zip(params, _firsts(params))]
    before = [p.detach().clone() for p in params]
    for step in range(2):
        for i, (p, r) in enumerate(zip(params, refs)):
            p.grad = None if i % 7 == 3 else _rand(p.shape, F32, step * 2000 + i)
            if p.grad is not None:
                r.step(p.grad)
            else:
                r.t += 1
        opt.step()
    for i, (p, r) in enumerate(zip(params, refs)):
        if i % 7 == 3:
            assert torch.equal(p.detach(), before[i])
            assert all(not opt.state[p][k].view(torch.uint8).any() for k in opt.state[p] if k != "step")
        else:
            _check_p(p, r, 2)
    live = [i for i in range(1500) if i % 7 != 3]
    _check_state(opt, [params[i] for i in live], [refs[i] for i in live], bits, 2)


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_share_a_group(optim, bits):
    kinds = [F32, BF16, F16, BF16, F32]
    params = [torch.nn.Parameter(_rand((300 + i,), t, i)) for i, t in enumerate(kinds)]
    opt = _make(optim, params, bits)
    refs = [Ref(p, bits, f) for p, f in zip(params, _firsts(params))]
    for i, (p, r) in enumerate(zip(params, refs)):
        p.grad = _rand(p.shape, p.dtype, 50 + i)
        r.step(p.grad)
    opt.step()
    for p, r in zip(params, refs):
        _check_p(p, r)
    _check_state(opt, params, refs, bits, 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts_and_alignment(optim, bits):
    flat = torch.nn.Parameter(_rand((5000,), F32, 1))
    views = [torch.nn.Parameter(v) for v in (flat.data[1:700], flat.data[703:1400].view(17, 41), flat.data[2000:2600])]
    cl = torch.nn.Parameter(_rand((16, 8, 3, 3), F32, 2).contiguous(memory_format=torch.channels_last))
    perm = torch.nn.Parameter(_rand((20, 30, 5), F32, 3).permute(2, 0, 1))
    half = torch.nn.Parameter(_rand((999,), BF16, 4)[3:])
    params = views + [cl, perm, half]
    opt = _make(optim, params, bits)
    around = flat.data.clone()
    refs = [Ref(p.detach().clone().as_strided((p.numel(),), (1,)) if p.is_contiguous() else
                p.data.as_strided((p.numel(),), (1,)), bits, f) for p, f in zip(params, _firsts(params))]
    for i, (p, r) in enumerate(zip(params, refs)):
        g = _rand(p.shape, p.dtype, 60 + i)          # contiguous, whatever the weight's order is
        p.grad = g
        r.step(torch.empty_like(p).copy_(g).as_strided((p.numel(),), (1,)) if not p.is_contiguous() else g)
    opt.step()
    for p, r in zip(params, refs):
        _check_p(p.data.as_strided((p.numel(),), (1,), p.storage_offset()), r)
    for a, b in ((0, 1), (700, 703), (1400, 2000), (2600, 5000)):
        assert torch.equal(flat.data[a:b], around[a:b])
    # the same gradients in the weights' own order give the same step
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    assert opt.state[cl]["exp_avg"].stride() == cl.stride()
    # an expanded gradient (a sum's)
    p = torch.nn.Parameter(_rand((40, 9), F32, 7))
    opt = _make(optim, [p], bits)
    r = Ref(p, bits)
    p.grad = torch.ones(1, 1, device="cuda").expand(40, 9)
    r.step(torch.ones(40, 9, device="cuda"))
    opt.step()
    _check_p(p, r)
    del again


@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_gradients(optim, bits):
    p = torch.nn.Parameter(_rand((4, 256), F32, 1))
    opt = _make(optim, [p], bits)
    r = Ref(p, bits)
    g = torch.zeros(4, 256, device="cuda")
    g[0] = _rand((256,), F32, 2) * torch.logspace(-15, 3, 256, device="cuda")   # 18 decades in a block
    g[1, 5] = 1e-18
    g[2] = 1e-25
    p.grad = g
    r.step(g)
    opt.step()
    assert p.isfinite().all()
    _check_p(p.detach()[[0, 1, 3]], _pick(r, [0, 1, 3]))
    if bits == 8:
        _check_state(opt, [p], [r], 8, 1)
        assert not ((opt.state[p]["exp_avg_sqrt"].float() == 0) & (g.abs() > 1e-18))[0].any()
    # no finite number: the element (32 bits) or its block (8 bits), and nothing else
    g = _rand((4, 256), F32, 3)
    g[1, 7], g[2, 9] = float("nan"), float("inf")
    p.grad = g
    opt.step()
    p.grad = _rand((4, 256), F32, 4)
    opt.step()
    bad = ~p.isfinite()
    assert not bad[[0, 3]].any() and bad[1, 7] and bad[2, 9]
    assert int(bad.sum()) == (2 if bits == 32 else 512)


def _pick(r, rows):
    out = Ref.__new__(Ref)
    out.t = r.t
    out.p, out.change = r.p.view(-1, 256)[rows].reshape(-1), r.change.view(-1, 256)[rows].reshape(-1)
    return out


def test_8_bit_moments_do_not_freeze(optim):
    """Under a constant gradient that drops to a tenth, v decays by 0.1 % a step.  The mean over 4096 elements of what 8 bits
    hold follows v to a hundredth (each is rounded once a step, up or down by at most an eighth of its value, with errors that
    cancel over the steps and the elements), where rounding to nearest would not move at all."""
    n = 4096
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = _make(optim, [p], 8, weight_decay=0.0)
    g0 = _rand((n,), F32, 1).abs() + 0.5
    m, v = torch.zeros(n, device="cuda").double(), torch.zeros(n, device="cuda").double()
    for step in range(400):
        g = g0 if step < 100 else g0 * 0.1
        p.grad = g
        opt.step()
        m, v = B1 * m + (1 - B1) * g.double(), B2 * v + (1 - B2) * g.double() ** 2
    s = opt.state[p]
    r = (s["exp_avg_sqrt"].float().view(-1, 256) * s["exp_avg_sqrt_scale"][:, None]).view(-1).double()
    assert abs(float((r / v.sqrt()).mean()) - 1) < 0.01
    held = (s["exp_avg"].float().view(-1, 256) * s["exp_avg_scale"][:, None]).view(-1).double()
    assert abs(float((held / m).mean()) - 1) < 0.02


@pytest.mark.parametrize("bits", [32, 8])
def test_scaler_hooks(optim, bits):
    params = [torch.nn.Parameter(_rand((500,), F32, i)) for i in range(3)]
    opt = _make(optim, params, bits)
    refs = [Ref(p, bits, f) for p, f in zip(params, _firsts(params))]
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    for step in range(4):
        for i, (p, r) in enumerate(zip(params, refs)):
            p.grad = _rand(p.shape, F32, 10 * step + i) * 1024.0
        if step == 1:
            params[1].grad[3] = float("inf")
        scale = float(scaler.scale(torch.ones(1, device="cuda")))
        before = [p.detach().clone() for p in params] + [t.clone() for t in opt.flat_state().values()]
        scaler.step(opt)
        scaler.update()
        if step == 1:
            after = [p.detach() for p in params] + list(opt.flat_state().values())
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) if a.dim() else torch.equal(a, b)
                       for a, b in zip(before, after))
        else:
            for p, r in zip(params, refs):
                r.step(p.grad, 1 / scale)
    for p, r in zip(params, refs):
        _check_p(p, r, 3)
    _check_state(opt, params, refs, bits, 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(optim, bits):
    def fresh():
        ps = [torch.nn.Parameter(_rand((700,), F32, 1)), torch.nn.Parameter(_rand((33, 9), BF16, 2))]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps

    lr = torch.tensor(LR, device="cuda")
    a, b = fresh(), fresh()
    oa, ob = _make(optim, a, bits), _make(optim, b, bits, lr=lr)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ob.step()
    for step in range(5):
        value = LR / (1 + step)
        lr.fill_(value)
        oa.param_groups[0]["lr"] = value
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad.copy_(_rand(p.shape, p.dtype, 30 + 2 * step + i))
            q.grad.copy_(p.grad)
        oa.step()
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())
    for x, y in zip(oa.flat_state().values(), ob.flat_state().values()):
        assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)
    assert int(ob.flat_state()["step"]) == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_other_stream_and_groups(optim, bits):
    ps = [torch.nn.Parameter(_rand((300,), F32, i)) for i in range(4)]
    opt = optim.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.5, "weight_decay": 0.0}], lr=LR, betas=(B1, B2), eps=EPS,
                      weight_decay=WD, state_bits=bits)
    refs = [Ref(p, bits, f) for p, f in zip(ps, _firsts(ps[:2]) * 2)]
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda e: 1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for p in ps:
            p.grad = p.detach() * 0.5
        opt.step()
    sched.step()
    torch.cuda.synchronize()
    for i, (p, r) in enumerate(zip(ps, refs)):
        r.step(r.p * 0.5, lr=LR if i < 2 else 0.5, wd=WD if i < 2 else 0.0)
        _check_p(p, r)


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints(optim, bits, tmp_path):
    def fresh(seed):
        return [torch.nn.Parameter(_rand((700,), F32, seed)),
                torch.nn.Parameter(_rand((8, 6, 3, 3), F32, seed + 1).contiguous(memory_format=torch.channels_last))]

    a = fresh(1)
    oa = _make(optim, a, bits)
    for step in range(3):
        for i, p in enumerate(a):
            p.grad = _rand(p.shape, F32, 10 * step + i)
        oa.step()
    torch.save(oa.state_dict(), tmp_path / "s.pt")
    b = [torch.nn.Parameter(p.detach().clone(memory_format=torch.preserve_format)) for p in a]
    ob = _make(optim, b, bits, lr=1.0)
    ob.load_state_dict(torch.load(tmp_path / "s.pt"))
    assert ob.param_groups[0]["lr"] == LR
    for p, q in zip(a, b):
        p.grad = _rand(p.shape, F32, 99)
        q.grad = p.grad.clone()
    oa.step()
    ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())
    for x, y in zip(oa.flat_state().values(), ob.flat_state().values()):
        assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)
    with pytest.raises(ValueError):
        _make(optim, fresh(1), 40 - bits).load_state_dict(oa.state_dict())
    with pytest.raises(ValueError):
        _make(optim, fresh(1)[:1], bits).load_state_dict(oa.state_dict())
    other = [torch.nn.Parameter(_rand((701,), F32, 1)), fresh(1)[1]]
    with pytest.raises(ValueError):
        _make(optim, other, bits).load_state_dict(oa.state_dict())
    plain = [fresh(1)[0], torch.nn.Parameter(_rand((8, 6, 3, 3), F32, 2))]
    oc = _make(optim, plain, bits)
    if bits == 8:
        with pytest.raises(ValueError):
            oc.load_state_dict(oa.state_dict())
    else:
        oc.load_state_dict(oa.state_dict())
        assert torch.equal(oc.state[plain[1]]["exp_avg"], oa.state[a[1]]["exp_avg"])


def test_step_refusals(optim):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4, 4, device="cuda")[:, :2])])
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float64))])
    p = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    opt = optim.AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    assert len(opt.param_groups) == 1
    with pytest.raises(ValueError), pytest.warns(UserWarning):
        optim.AdamW([p, p])
    p.grad = torch.ones(4, 4, device="cuda")
    p.data = torch.zeros(8, 4, device="cuda")[::2]
    with pytest.raises(ValueError):
        opt.step()
    p.data = torch.zeros(5, 5, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
    p = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    opt = optim.AdamW([p])
    p.grad = torch.ones(4, 4, device="cuda").to_sparse()
    with pytest.raises(ValueError):
        opt.step()
    opt.zero_grad()
    opt.step()                                # nothing to do
    assert int(opt.flat_state()["step"]) == 0
    opt = optim.AdamW([p], lr=torch.tensor(-1.0))
    p.grad = torch.ones(4, 4, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
    import copy
    with pytest.raises(TypeError):
        copy.deepcopy(opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_2_to_the_31_elements(optim, bits):
    n = 2 ** 31 + 2 ** 20 + 77
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(300, dtype=BF16, device="cuda"))
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    tail = 1000
    with torch.no_grad():
        p[-tail:] = _rand((tail,), BF16, 1)
    p.grad[-tail:] = _rand((tail,), BF16, 2)
    q.grad = _rand((300,), BF16, 3)
    opt = _make(optim, [p, q], bits)
    # the tail's blocks as a tensor of its own that begins at the same place
    start = (n - tail) // 256 * 256
    ref_p = torch.zeros(n - start, dtype=BF16, device="cuda")
    ref_p[-tail:] = p.detach()[-tail:]
    ref, ref_q = Ref(ref_p, bits, start), Ref(q, bits, -(-n // 256) * 256)
    g = torch.zeros(n - start, device="cuda")
    g[-tail:] = p.grad[-tail:].float()
    ref.step(g)
    ref_q.step(q.grad)
    opt.step()
    _check_p(p.detach()[start:], ref)
    _check_p(q, ref_q)
    s = opt.state[p]
    if bits == 8:
        assert torch.equal(s["exp_avg"][start:].double(), ref.m8.view(-1)[:n - start])
        assert torch.equal(s["exp_avg_sqrt_scale"][start // 256:].double(), ref.rs.view(-1))
    assert not s["exp_avg"][:start].view(torch.uint8).any() and not p.detach()[:start].any()


# ---- the operators together -------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_training_of_quantised_layers(ops, optim, bits):
    """Two int8 layers, their gradients and the optimizer's step, captured into a graph and replayed, against the same steps
    one by one; then the trained weights prepared for serving."""
    def model():
        return [torch.nn.Parameter(_rand((256, 128), F32, 1, 0.1)), torch.nn.Parameter(torch.zeros(256, device="cuda")),
                torch.nn.Parameter(_rand((10, 256), F32, 2, 0.1)), torch.nn.Parameter(torch.zeros(10, device="cuda"))]

    def loss_of(w, x, y):
        h = torch.relu(ops.int8_linear(x, w[0], w[1]))
        return torch.nn.functional.cross_entropy(ops.int8_linear(h, w[2], w[3]), y)

    x, y = _rand((64, 128), F32, 5), torch.randint(0, 10, (64,), device="cuda")
    a, b = model(), model()
    oa, ob = _make(optim, a, bits), _make(optim, b, bits)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                # warm-up on a side stream; its graph is dropped before the capture
        loss_of(b, x, y).backward()
    torch.cuda.current_stream().wait_stream(s)
    for p in b:
        p.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for p in b:
            p.grad = None
        loss = loss_of(b, x, y)
        loss.backward()
        ob.step()
    for step in range(6):
        for p in a:
            p.grad = None
        ref = loss_of(a, x, y)
        ref.backward()
        oa.step()
        graph.replay()
        assert torch.equal(ref.detach(), loss.detach())
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())
    assert int(ob.flat_state()["step"]) == 6
    with torch.no_grad():
        w1, w2 = ops.int8_quantize(a[0]), ops.int8_quantize(a[2])
        served = ops.int8_linear(torch.relu(ops.int8_linear(x, w1, a[1])), w2, a[3])
        assert torch.equal(served, ops.int8_linear(torch.relu(ops.int8_linear(x, a[0], a[1])), a[2], a[3]))
    assert ops.int8_status() == 0


@pytest.mark.parametrize("name, bits", [("adamw", 32), ("adamw8", 8)])
def test_optimizer_of_the_training_driver(ops, optim, name, bits):
    """The optimizer that the training driver makes by name, in a step as the fp16 loop takes it: channels_last model,
    autocast, loss scaling, gradients in the weights' memory format or not."""
    import dataclasses

    from rexsc_b200.frontend import train

    wl = dataclasses.replace(train.WORKLOADS["resnet18_or2_L32"], optimizer=name)
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 16, 3), torch.nn.BatchNorm2d(16), torch.nn.ReLU(), torch.nn.Conv2d(16, 8, 3),
                                torch.nn.Flatten(), torch.nn.Linear(8 * 12 * 12, 10)).cuda().to(memory_format=torch.channels_last)
    opt = train.make_optimizer(wl, model, lr=1e-3)
    assert isinstance(opt, optim.AdamW) and isinstance(opt, torch.optim.Optimizer)
    assert opt.flat_state()["exp_avg"].dtype == (F32 if bits == 32 else torch.float8_e4m3fn)
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 10)
    x = _rand((4, 3, 16, 16), F32, 1).contiguous(memory_format=torch.channels_last)
    y = torch.randint(0, 10, (4,), device="cuda")
    before = [p.detach().clone() for p in model.parameters()]
    for _ in range(3):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=F16):
            loss = torch.nn.functional.cross_entropy(model(x), y)
        scaler.scale(loss).backward()
        scaler.step(opt)
        scaler.update()
    assert int(opt.flat_state()["step"]) == 3
    for p, q in zip(model.parameters(), before):
        assert p.isfinite().all() and not torch.equal(p.detach(), q)
    with pytest.raises(ValueError):
        train.make_optimizer(dataclasses.replace(wl, optimizer="rmsprop"), model)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_counts_as_a_write(optim, bits):
    """A graph that still needs the weights of before a step raises, as after any write in place."""
    p, q, still = (torch.nn.Parameter(_rand((300,), seed=i)) for i in range(3))
    opt = optim.AdamW([p, q, still], state_bits=bits)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    later, other = (p * p).sum(), (still * still).sum()
    versions = p._version, q._version, still._version
    opt.step()
    assert p._version > versions[0] and q._version > versions[1] and still._version == versions[2]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        later.backward()
    other.backward()


def test_parameters_that_share_memory(optim):
    flat = torch.zeros(1000, device="cuda")
    halves = [torch.nn.Parameter(flat[:500]), torch.nn.Parameter(flat[500:])]
    opt = optim.AdamW(halves)
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(flat[499:501])]})
    assert len(opt.param_groups) == 1
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(flat), torch.nn.Parameter(flat.view(10, 100))])
    for p in halves:
        p.grad = torch.ones_like(p)
    opt.step()
    assert (flat == flat[0]).all() and flat[0] != 0


@pytest.mark.parametrize("bits", [32, 8])
def test_strides_of_single_elements_do_not_matter(optim, bits):
    """The same places with other strides where a dimension has one element: no new layout, for weights and for gradients."""
    a, b = (torch.nn.Parameter(_rand((6, 1, 3, 3))) for _ in range(2))
    oa, ob = optim.AdamW([a], state_bits=bits), optim.AdamW([b], state_bits=bits)
    a.grad, b.grad = _rand((6, 1, 3, 3), seed=1), _rand((6, 1, 3, 3), seed=1).as_strided((6, 1, 3, 3), (9, 1, 3, 1))
    b.data = b.data.as_strided((6, 1, 3, 3), (9, 1, 3, 1))
    assert a.stride() != b.stride()
    oa.step()
    ob.step()
    assert torch.equal(a, b)
