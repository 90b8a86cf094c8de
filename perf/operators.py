"""The operators of quantised layers in training and serving, as cases to measure.

Kinds (``"kind"`` of a case):

  serve   ``ops.int8_linear(x, weights, bias)`` with weights quantised once per output channel: tokens are quantised per
          row, multiplied in 8-bit integers and scaled back
  train   ``ops.int8_linear(x, w, bias)`` on float weights, forward and backward: all three products in 8-bit integers
  adamw   ``optim.AdamW(...).step()`` over a list of parameters, moments in 32 or in 8 bits

``own`` false: the operators in their plain form, elementary torch operations.  ``own`` true: the framework's calls.

A row is quantised as  s = max|x| / 127  (held in 32 bits),  q = x / (max|x| / 127)  rounded to the nearest whole number,
ties to even; an all-zero row has s = 0.  Values on the border between two whole numbers decide by the exact quotient, so
the plain form takes the quotients of 32-bit inputs in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 256                     # elements of 8-bit moments that share a scale
BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.999, 1e-8, 1e-3, 1e-2
LOSS_SCALE = 65536.0            # initial scale of torch.amp.GradScaler


# ---- cases ----------------------------------------------------------------------------------------------------
def _linear(kind, m, k, n, dtype, wtype, bias, name=None):
    case = dict(kind=kind, m=m, k=k, n=n, dtype=dtype, wtype=wtype, bias=bias)
    return dict(case, name=name) if name else case


def _adamw(bits, model, total, tensors, dtype, gtype, scaled, name=None):
    """``model``: the shapes of a network of the framework's workloads, or "" for ``tensors`` tensors of ``total`` elements."""
    case = dict(kind="adamw", bits=bits, model=model, total=total, tensors=tensors, dtype=dtype, gtype=gtype, scaled=scaled)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token through a square layer with prepared weights: reading the weights is all there is
        _linear("serve", 1, 4096, 4096, "bf16", "bf16", False, "serve_1x4096x4096"),
        # a few tokens, sizes that fill no tile and no 16-byte vector
        _linear("serve", 13, 2051, 5003, "f16", "f32", True, "serve_13x2051x5003"),
        # the classifier of ResNet-18 at its training batch, evaluated
        _linear("serve", 256, 512, 1000, "f32", "f32", True, "serve_256x512x1000"),
        # a long prompt through a wide layer: the tensor cores bound it
        _linear("serve", 8192, 8192, 8192, "bf16", "bf16", False, "serve_8192x8192x8192"),
        # a training step of the same classifier
        _linear("train", 256, 512, 1000, "f32", "f32", True, "train_256x512x1000"),
        # ragged batch of tokens, sizes odd in every direction
        _linear("train", 1537, 1111, 2049, "f16", "f32", True, "train_1537x1111x2049"),
        # a batch of sequences through a square layer, weights in 16 bits
        _linear("train", 8192, 4096, 4096, "bf16", "bf16", False, "train_8192x4096x4096"),
        # the optimizer step of TinyConv: four convs and little else, launch latency counts
        _adamw(32, "tinyconv", 0, 0, "f32", "f32", False, "adamw32_tinyconv"),
        # ResNet-18 under a GradScaler, as the fp16 training loop steps it
        _adamw(32, "resnet18", 0, 0, "f32", "f32", True, "adamw32_resnet18"),
        # the same with moments in 8 bits
        _adamw(8, "resnet18", 0, 0, "f32", "f32", True, "adamw8_resnet18"),
        # layers of a large model: 32-bit weights and moments; 16-bit weights and 8-bit moments
        _adamw(32, "", 134217728, 24, "f32", "bf16", False, "adamw32_134M"),
        _adamw(8, "", 134217728, 24, "bf16", "bf16", False, "adamw8_134M"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("serve", "serve", "train", "adamw", "adamw"))
    if kind == "adamw":
        return _adamw(rng.choice((8, 32)), "", _log(rng, 1 << 14, 134217728), _log(rng, 1, 200),
                      rng.choice(("f32", "f32", "bf16", "f16")), rng.choice(("f32", "bf16", "f16")), rng.random() < 0.5)
    m, k, n = _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 8, 8192)
    if kind == "train":
        m, k, n = max(m, 2), _log(rng, 16, 4096), _log(rng, 8, 4096)
    if rng.random() < 0.5:      # sizes as layers have them
        k, n = -(-k // 64) * 64, -(-n // 64) * 64
    return _linear(kind, m, k, n, rng.choice(("f32", "f16", "bf16")), rng.choice(("f32", "bf16", "f16")), rng.random() < 0.5)


# ---- shapes of the networks -----------------------------------------------------------------------------------
def _conv_bn(co, ci, k):
    return [(co, ci, k, k), (co,), (co,)]


def _resnet18():
    shapes = _conv_bn(64, 3, 7)
    cin = 64
    for stage, co in enumerate((64, 128, 256, 512)):
        for block in range(2):
            shapes += _conv_bn(co, cin if block == 0 else co, 3) + _conv_bn(co, co, 3)
            if block == 0 and stage:
                shapes += _conv_bn(co, cin, 1)
        cin = co
    return shapes + [(1000, 512), (1000,)]


def _tinyconv():
    return _conv_bn(32, 3, 5) + _conv_bn(32, 32, 5) + _conv_bn(64, 32, 5) + [(10, 64, 4, 4), (10,), (10,)]


def _shapes(case):
    if case["model"]:
        return {"resnet18": _resnet18, "tinyconv": _tinyconv}[case["model"]]()
    # tensors of very different sizes: every second one a small vector (a bias, a norm's weight)
    total, count = case["total"], case["tensors"]
    large = (count + 1) // 2
    small = [(1 + (37 * i) % 1000,) for i in range(count - large)]
    left = max(large, total - sum(s[0] for s in small))
    weights = [1 + (i % 3) for i in range(large)]
    return [(max(1, left * w // sum(weights)),) for w in weights] + small


def _places(shapes):
    """(start, elements) of each tensor in flat storage where every one begins on a block of its own, and the length."""
    places, at = [], 0
    for s in shapes:
        n = math.prod(s)
        places.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return places, at


# ---- inputs ---------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale)


def _linear_inputs(case, seed):
    g, m, k, n = _gen(seed), case["m"], case["k"], case["n"]
    x = _normal(g, (m, k))
    x[:, :: max(1, k // 7)] *= 12.0              # a few channels far above the others, as activations have them
    if m > 20:
        x[5::17] = 0                             # tokens of a padded batch
    w = _normal(g, (n, k), 1 / math.sqrt(k))
    made = {"x": x.to(DTYPES[case["dtype"]]), "w": w.to(DTYPES[case["wtype"]]),
            "bias": _normal(g, (n,)) if case["bias"] else None}
    if case["kind"] == "train":
        made["dy"] = _normal(g, (m, n), 1e-2).to(DTYPES[case["dtype"]])
    return made


def _adamw_inputs(case, seed):
    """Flat storage of weights and gradients, the tensors' places in it, moments after some hundred steps and their count."""
    g = _gen(seed)
    shapes = _shapes(case)
    places, total = _places(shapes)
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for at, n in places:
        live[at:at + n] = True
    t = 100 + int(seed) % 900
    size = torch.exp(_normal(g, (total // BLOCK, 1), 2.0)) * 1e-3   # gradients of different magnitude
    grad = (_normal(g, (total // BLOCK, BLOCK)) * size).view(-1) * live
    m = (_normal(g, (total // BLOCK, BLOCK), 0.3) * size).view(-1) * live
    v = ((0.5 + torch.rand(total // BLOCK, BLOCK, generator=g, device="cuda")) * size).view(-1).square() * live
    grad = grad * (LOSS_SCALE if case["scaled"] else 1.0)
    if case["gtype"] == "f16":
        grad = grad.clamp_(-6e4, 6e4)
    made = {"p": (_normal(g, (total,), 0.05) * live).to(DTYPES[case["dtype"]]), "g": grad.to(DTYPES[case["gtype"]]),
            "shapes": shapes, "places": places, "t": t, "m": m, "v": v}
    if case["bits"] == 8:
        for name, x in (("m", m), ("r", v.sqrt())):
            s = x.view(-1, BLOCK).abs().amax(1) / 448
            code = (x.view(-1, BLOCK) / s.clamp(min=1e-30).unsqueeze(1)).clamp(-448, 448).to(torch.float8_e4m3fn)
            made[name + "8"], made[name + "s"] = code.view(-1), s
        del made["m"], made["v"]
    return made


def _views(flat, made):
    return [flat[at:at + n].view(s) for s, (at, n) in zip(made["shapes"], made["places"])]


def prepare(case, seed):
    if case["kind"] == "adamw":
        made = _adamw_inputs(case, seed)
        state = dict(case=case, p=made["p"], g=made["g"], t=made["t"])
        if case["scaled"]:
            state["scale"], state["inf"] = (torch.full((), v, device="cuda") for v in (LOSS_SCALE, 0.0))
        if own:
            from rexsc_b200 import optim

            params = [torch.nn.Parameter(v) for v in _views(made["p"], made)]
            for p, v in zip(params, _views(made["g"], made)):
                p.grad_dtype = None
                p.grad = v
            opt = optim.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"])
            flat = opt.flat_state()
            flat["step"].fill_(made["t"])
            if case["bits"] == 8:
                flat["exp_avg"].copy_(made["m8"]), flat["exp_avg_scale"].copy_(made["ms"])
                flat["exp_avg_sqrt"].copy_(made["r8"]), flat["exp_avg_sqrt_scale"].copy_(made["rs"])
            else:
                flat["exp_avg"].copy_(made["m"]), flat["exp_avg_sq"].copy_(made["v"])
            if case["scaled"]:  # what GradScaler.step hands to an optimizer that unscales by itself
                opt.grad_scale, opt.found_inf = state["scale"], state["inf"]
            state.update(opt=opt, flat=flat)
        else:
            state.update({k: made[k] for k in ("m", "v", "m8", "ms", "r8", "rs") if k in made})
        return state
    made = _linear_inputs(case, seed)
    state = dict(case=case, **made)
    if case["kind"] == "serve":
        w = state.pop("w")
        if own:
            from rexsc_b200 import ops

            state["weights"] = ops.int8_quantize(w)
        else:
            state["qw"], state["sw"] = _rows(w)
    elif own:
        for name in ("x", "w", "bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------
def _over(a, b):
    """a / b with one rounding; torch divides by a number, or a number, with two (it multiplies by a reciprocal)."""
    like = a if isinstance(a, torch.Tensor) else b
    return torch.as_tensor(a, device=like.device).expand_as(like) / torch.as_tensor(b, device=like.device).expand_as(like)


def _rows(x):
    """Whole numbers (in 8 bits) and scales of the rows of ``x``."""
    a = x.abs().amax(1, keepdim=True)
    q = (x.double() * 127 / a.double().where(a > 0, 1.0)).round()
    return q.to(torch.int8), _over(a.float(), 127.0).squeeze(1)


def _product(qa, qb):
    """Sums of products of whole numbers; they pass 2^24, so they are taken in 64 bits."""
    return (qa.double() @ qb.double().t()).float()


def _plain_forward(qx, sx, qw, sw, bias, dtype):
    y = _product(qx, qw) * sx.unsqueeze(1) * sw
    return (y if bias is None else y + bias).to(dtype)


def _plain_train(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    (qx, sx), (qw, sw) = _rows(x), _rows(w)
    y = _plain_forward(qx, sx, qw, sw, s["bias"], x.dtype)
    qg, sg = _rows(dy.float() * sw)
    qh, sh = _rows((dy.float() * sx.unsqueeze(1)).t())
    dx = (_product(qg, qw.t()) * sg.unsqueeze(1)).to(x.dtype)
    dw = (_product(qh, qx.t()) * sh.unsqueeze(1)).to(w.dtype)
    return [y, dx, dw] + ([] if s["bias"] is None else [dy.double().sum(0).float()])


def _threshold(total, t):
    """Rounding thresholds in [0, 2^32): equidistributed over the places of one step and over the steps of one place."""
    at = torch.arange(total, device="cuda", dtype=torch.int64)
    return (at * 0xC13FA9A9 + t * 0x9E3779B9) & 0xFFFFFFFF


def _to_e4m3(y, u, least):
    """``y`` >= 0 as e4m3: up where the fraction that is cut off and ``u`` (20 bits) make one step, never below ``least``."""
    normal = ((y.view(torch.int32) + u.int()) & ~0xFFFFF).view(torch.float32)
    small = (y * 512 + u.float() * 2.0 ** -20).floor() / 512
    return torch.where(y < 2.0 ** -6, small, normal).clamp(max=448.0).maximum(least)


def _plain_store(x, u, floor):
    """Codes and scales of a moment; ``floor``: what is not 0 is not stored as 0."""
    a = x.view(-1, BLOCK).abs().amax(1, keepdim=True)
    fine = a >= 2.0 ** -100
    y = x.abs().view(-1, BLOCK) * _over(448.0, a).where(fine, 0.0)
    least = ((y > 0) * floor * 2.0 ** -9).view(-1)
    code = _to_e4m3(y.view(-1), u, least) * x.sign()
    return code.to(torch.float8_e4m3fn), _over(a, 448.0).where(fine, 0.0).view(-1)


def _plain_adamw(s):
    s["t"] += 1
    t, g = s["t"], s["g"].float()
    if "scale" in s:
        g = g * (1 / s["scale"])
    if s["case"]["bits"] == 8:
        m = (s["m8"].float().view(-1, BLOCK) * s["ms"].unsqueeze(1)).view(-1)
        v = (s["r8"].float().view(-1, BLOCK) * s["rs"].unsqueeze(1)).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    r = v.sqrt()
    p = s["p"].float() * (1 - LR * DECAY) - LR / (1 - BETA1 ** t) * m / (r / math.sqrt(1 - BETA2 ** t) + EPS)
    s["p"] = p.to(s["p"].dtype)
    if s["case"]["bits"] == 32:
        s["m"], s["v"] = m, v
        return [s["p"], m, v]
    u = _threshold(m.numel(), t)
    s["m8"], s["ms"] = _plain_store(m, u >> 12, 0.0)
    s["r8"], s["rs"] = _plain_store(r, (u ^ 0xFFFFFFFF) >> 12, 1.0)
    return [s["p"], s["m8"], s["ms"], s["r8"], s["rs"]]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        if kind == "adamw":
            return _plain_adamw(state)
        if kind == "train":
            return _plain_train(state)
        qx, sx = _rows(state["x"])
        return _plain_forward(qx, sx, state["qw"], state["sw"], state["bias"], state["x"].dtype)
    if kind == "adamw":
        state["opt"].step()
        flat = state["flat"]
        return [state["p"]] + [flat[k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sqrt", "exp_avg_sqrt_scale") if k in flat]
    from rexsc_b200 import ops

    if kind == "serve":
        return ops.int8_linear(state["x"], state["weights"], state["bias"])
    y = ops.int8_linear(state["x"], state["w"], state["bias"])
    wanted = [state[k] for k in ("x", "w", "bias") if state[k] is not None]
    return [y.detach(), *torch.autograd.grad(y, wanted, state["dy"])]


# ---- the definition in 64 bits --------------------------------------------------------------------------------
def _fl32(x):
    """A value that the operator holds in 32 bits, in 64."""
    return x.float().double()


def _exact_quantise(x, dim):
    """Whole numbers, and scales as the operator holds them, along ``dim`` of ``x`` (64 bits)."""
    most = x.abs().max(dim, keepdim=True).values
    step = most / 127
    q = torch.where(most > 0, x * 127 / torch.where(most > 0, most, torch.ones_like(most)), torch.zeros_like(x))
    return torch.round(q), _fl32(step)


def _exact_linear(case, seed):
    made = _linear_inputs(case, seed)
    x, w = made["x"].double(), made["w"].double()
    qx, sx = _exact_quantise(x, 1)
    qw, sw = _exact_quantise(w, 1)
    y = torch.einsum("mk,nk->mn", qx, qw) * (sx * sw.t())
    if made["bias"] is not None:
        y += made["bias"].double()
    if case["kind"] == "serve":
        return y
    dy = made["dy"].double()
    qg, sg = _exact_quantise(_fl32(dy * sw.t()), 1)
    qh, sh = _exact_quantise(_fl32(dy * sx), 0)
    out = [y, torch.einsum("mn,nk->mk", qg, qw) * sg, torch.einsum("mn,mk->nk", qh, qx) * sh.t()]
    return out + ([dy.sum(0)] if made["bias"] is not None else [])


def _exact_code(y, u, least):
    """``y`` >= 0 (64 bits) cut to four significant bits (steps of 2^-9 at the least), up by ``u`` / 2^20 of a step."""
    exponent = torch.frexp(y).exponent - 1
    step = torch.exp2((exponent - 3).clamp(min=-9).double())
    code = torch.floor(y / step + u.double() / 2 ** 20) * step
    return torch.minimum(code, torch.full_like(code, 448.0)).maximum(least)


def _exact_store(x, u, floor):
    """The definition cuts a moment that it holds in 32 bits, in units of a scale that it holds in 32 bits."""
    rows = x.reshape(-1, BLOCK)
    most = rows.abs().max(1, keepdim=True).values
    live = most >= 2.0 ** -100
    per = torch.where(live, _fl32(448 / most), torch.zeros_like(most))
    y = _fl32(rows.abs() * per).reshape(-1)
    least = torch.where(y > 0, floor * 2.0 ** -9, 0.0).double()
    return _exact_code(y, u, least) * torch.sign(x), torch.where(live, _fl32(most / 448), torch.zeros_like(most)).reshape(-1)


def _exact_adamw(case, seed):
    made = _adamw_inputs(case, seed)
    t = made["t"] + 1
    g = made["g"].double()
    if case["scaled"]:
        g = g / LOSS_SCALE
    if case["bits"] == 8:
        # moments that leave as 8 bits are decided by the values that the operator holds in 32 bits on the way
        m = _fl32(made["m8"].double().reshape(-1, BLOCK) * made["ms"].double().unsqueeze(1)).reshape(-1)
        v = _fl32(_fl32(made["r8"].double().reshape(-1, BLOCK) * made["rs"].double().unsqueeze(1)).reshape(-1) ** 2)
        b1, c1, b2, c2 = (float(torch.tensor(c, dtype=torch.float32)) for c in (BETA1, 1 - BETA1, BETA2, 1 - BETA2))
        m = _fl32(_fl32(b1 * m) + _fl32(c1 * g))
        r = _fl32(torch.sqrt(_fl32(_fl32(b2 * v) + _fl32(c2 * _fl32(g * g)))))
    else:
        m = made["m"].double() * BETA1 + g * (1 - BETA1)
        v = made["v"].double() * BETA2 + g ** 2 * (1 - BETA2)
        r = torch.sqrt(v)
    p = made["p"].double()
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (r / math.sqrt(1 - BETA2 ** t) + EPS)
    if case["bits"] == 32:
        return [p, m, v]
    at = torch.arange(m.numel(), device="cuda", dtype=torch.int64)
    u = (at * 3242174889 + t * 2654435769) % (1 << 32)
    m8, ms = _exact_store(m, u // 4096, 0.0)
    r8, rs = _exact_store(r, ((1 << 32) - 1 - u) // 4096, 1.0)
    return [p, m8, ms, r8, rs]


def exact(case, seed):
    return _exact_adamw(case, seed) if case["kind"] == "adamw" else _exact_linear(case, seed)


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def work(case):
    if case["kind"] == "adamw":
        shapes = _shapes(case)
        n = sum(math.prod(s) for s in shapes)
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK      # two, read and written, with their scales
        return dict(bytes=int(n * (2 * SIZE[case["dtype"]] + SIZE[case["gtype"]] + moments)), flops=20 * n)
    m, k, n = case["m"], case["k"], case["n"]
    size, wsize, bias = SIZE[case["dtype"]], SIZE[case["wtype"]], 4 * n * case["bias"]
    if case["kind"] == "serve":
        return dict(bytes=size * (m * k + m * n) + n * k + 4 * n + bias, flops=2 * m * n * k)
    # x, w, dy read; y, dx, dw, db written
    return dict(bytes=size * 2 * (m * k + m * n) + wsize * 2 * n * k + 2 * bias, flops=6 * m * n * k)
