"""Linear layers in 8-bit integers against their definition in 64 bits.

The integers and the scales have to be equal.  The sums of products are exact, so that an fp32 output is off by the three
roundings of the sum and its two scalings (2^-24 each, relative) and one more with a bias; an output in 16 bits by half a step
of its type on top."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(shape, dtype=F32, seed=0, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed), device="cuda") * scale).to(dtype)


def _quant(x, dim=1):
    """Integers and scales (64 bits) along ``dim``; a row with an infinity or a NaN is 0 with the scale NaN."""
    x = x.double()
    a = x.abs().amax(dim, keepdim=True)
    fine = a.isfinite()
    a0 = torch.where(fine & (a > 0), a, 1.0)
    q = torch.where(fine, (x.nan_to_num(0, 0, 0) * 127 / a0).round(), 0.0)
    s = torch.where(fine, a.float().nan_to_num(0, 0, 0) / torch.full_like(a, 127.0).float(), float("nan"))
    return q, s.double().squeeze(dim)


def _allowed(ref, dtype, parts):
    """Bound of the error of ``ref`` rounded to ``dtype``; ``parts``: magnitude of what was added up in fp32."""
    info = torch.finfo(dtype)
    fp32 = 4 * 2.0 ** -24 * parts + 2.0 ** -149
    return fp32 if dtype == F32 else fp32 + (ref.abs() + fp32) * info.eps / 2 + info.smallest_normal * info.eps / 2


def _check(got, ref, parts=None):
    parts = ref.abs() if parts is None else parts
    err = (got.double() - ref).abs()
    bad = err > _allowed(ref, got.dtype, parts)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(err.max())} where {float(parts.max())} is the largest"


def _linear_ref(x, w, bias=None):
    (qx, sx), (qw, sw) = _quant(x), _quant(w)
    y = (qx @ qw.t()) * sx[:, None] * sw
    parts = y.abs()
    if bias is not None:
        y = y + bias.double()
        parts = parts + bias.double().abs()
    return y, parts


# ---- quantisation -----------------------------------------------------------------------------------------------
SIZES = [(1, 1), (1, 16), (3, 17), (2, 127), (130, 129), (5, 1000), (9, 1024), (7, 1025), (2, 2048), (3, 4096), (2, 4104),
         (300, 136), (2, 8192), (2, 8199), (1, 20011), (257, 640)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, cols", SIZES)
def test_quantised_integers_and_scales_are_exact(ops, rows, cols, dtype):
    x = _rand((rows, cols), dtype, rows + cols)
    m = ops.int8_quantize(x)
    q, s = _quant(x)
    assert m.shape == (rows, cols)
    assert torch.equal(m.values().double(), q) and torch.equal(m.scale.double(), s)
    # what pads the tiles is zero: it is multiplied with the padding of the other operand
    assert int(m.data.view(torch.int8).ne(0).sum()) == int(q.ne(0).sum())
    assert torch.equal(m.dequantize(), q.float() * s.float()[:, None])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_values_on_the_border_between_two_integers(ops, dtype):
    # multiples of half a step of rows whose largest magnitude is 127 (exact in every type), and their neighbours
    half = torch.arange(-254, 255, device="cuda").float() / 2
    rows = [half]
    up = torch.nextafter(half, torch.full_like(half, 1e9))
    down = torch.nextafter(half, torch.full_like(half, -1e9))
    rows += [up.clamp(-127, 127), down.clamp(-127, 127)]
    x = torch.stack(rows).to(dtype)
    x[:, 0] = 127
    x = torch.cat([x, x / 64, x * 32, (x.float() * 2.0 ** -20).to(dtype)])
    m = ops.int8_quantize(x)
    q, s = _quant(x)
    assert torch.equal(m.values().double(), q) and torch.equal(m.scale.double(), s)


def test_rows_of_extreme_values(ops):
    x = torch.zeros(12, 300, device="cuda")
    x[1, 7] = 1.0
    x[2] = 3e38 * torch.linspace(-1, 1, 300, device="cuda")
    x[3] = 1e-30 * torch.linspace(-1, 1, 300, device="cuda")
    x[4] = 1e-37 * torch.linspace(-1, 1, 300, device="cuda")
    x[5] = 1e-42 * torch.linspace(-1, 1, 300, device="cuda")
    x[6, 3] = float("inf")
    x[7, 4] = float("nan")
    x[7, 5] = float("inf")
    x[8, 0] = -float("inf")
    x[9, 299] = -5.0
    x[10] = torch.finfo(F32).min
    x[11] = torch.finfo(F32).tiny
    m = ops.int8_quantize(x)
    q, s = _quant(x)
    assert torch.equal(m.values().double(), q)
    assert torch.equal(m.scale.isnan(), s.isnan()) and torch.equal(m.scale.nan_to_num().double(), s.nan_to_num())
    y = ops.int8_linear(x, ops.int8_quantize(_rand((40, 300))))
    assert y[[6, 7, 8]].isnan().all() and not y[[0, 1, 2, 3, 4, 5, 9, 10, 11]].isnan().any()
    assert (y[0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_and_unaligned_rows(ops, dtype):
    base = _rand((40, 700), dtype)
    flat = _rand((9 * 333 + 5,), dtype)
    views = [base[:, :333], base[:, 3:520], base[::3, 8:648], base[:20].t(), flat[5:].view(9, 333), base[:, 4:5],
             base[:1].expand(6, 700), base[:, :1].expand(40, 64), base.flip(0)]
    for v in views:
        m = ops.int8_quantize(v)
        q, s = _quant(v)
        assert torch.equal(m.values().double(), q) and torch.equal(m.scale.double(), s)


def test_pack_and_unpack_plain_integers(ops):
    for rows, cols in [(1, 1), (130, 257), (128, 128), (5, 1003)]:
        v = torch.randint(-128, 128, (rows, cols), generator=_gen(), device="cuda").to(torch.int8)
        s = torch.rand(rows, device="cuda")
        m = ops.Int8Matrix.from_values(v, s)
        assert torch.equal(m.values(), v) and torch.equal(m.scale, s)
    t = ops.Int8Matrix.from_values(v.t(), torch.rand(cols, device="cuda"))
    assert torch.equal(t.values(), v.t())


# ---- products ---------------------------------------------------------------------------------------------------
PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 1000, 512), (3, 129, 33), (16, 128, 1024), (17, 257, 130), (33, 70, 4096),
            (64, 640, 640), (65, 256, 4100), (128, 512, 256), (130, 300, 1500), (256, 256, 128), (257, 513, 385),
            (300, 1000, 512), (700, 1300, 900), (1024, 520, 2050)]


@pytest.mark.parametrize("kernel", ["split", "pair", "auto"])
@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_sums_of_products_are_exact(ops, m, n, k, kernel):
    a = torch.randint(-128, 128, (m, k), generator=_gen(1), device="cuda").to(torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=_gen(2), device="cuda").to(torch.int8)
    ones_m, ones_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    ops.set_int8_kernel(kernel)
    try:
        y = ops.int8_matmul(ops.Int8Matrix.from_values(a, ones_m), ops.Int8Matrix.from_values(b, ones_n))
    finally:
        ops.set_int8_kernel("auto")
    assert ops.int8_status() == 0
    assert torch.equal(y, (a.double() @ b.double().t()).float())


@pytest.mark.parametrize("m, n, k", [(2600, 2700, 300), (5000, 600, 1100), (300, 20000, 130), (260, 260, 20000), (40, 300, 40000),
                                     (20000, 130, 128)])
def test_many_tiles_and_long_contractions(ops, m, n, k):
    # more output tiles than CTAs, rings of stages filled many times over, several products' accumulators in turn
    a = torch.randint(-128, 128, (m, k), generator=_gen(1), device="cuda").to(torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=_gen(2), device="cuda").to(torch.int8)
    ma = ops.Int8Matrix.from_values(a, torch.ones(m, device="cuda"))
    mb = ops.Int8Matrix.from_values(b, torch.ones(n, device="cuda"))
    ref = (a.double() @ b.double().t()).float()
    for kernel in ("split", "pair", "auto"):
        ops.set_int8_kernel(kernel)
        y = ops.int8_matmul(ma, mb)
        ops.set_int8_kernel("auto")
        assert torch.equal(y, ref), kernel
    assert ops.int8_status() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n, k", [(1, 1), (130, 9), (300, 128), (1000, 515), (77, 2000), (4096, 4096), (129, 33000)])
def test_a_few_tokens(ops, n, k, dtype):
    """Up to 32 tokens are quantised by the product's kernel where they are few values; forcing the other kernel quantises them
    with a launch of their own.  Both are the same integers and sums."""
    base = _rand((33, k + 3), dtype, 1)
    base[4] = 0
    base[6] = float("nan")
    base[6, 3] = float("inf")
    base[9] *= 1e-30 if dtype != F16 else 1e-6
    w = ops.int8_quantize(_rand((n, k), F32, 2, k ** -0.5))
    bias = _rand((n,), BF16, 3)
    for x in (base[:, :k], base[:, 3:], base[:, 1:k + 1].contiguous()):
        for m in (1, 2, 3, 4, 5, 8, 13, 16, 17, 24, 31, 32, 33):
            y = ops.int8_linear(x[:m], w, bias)
            ops.set_int8_kernel("pair")
            ref = ops.int8_linear(x[:m], w, bias)
            ops.set_int8_kernel("auto")
            assert torch.equal(y.nan_to_num(7.0), ref.nan_to_num(7.0)) and torch.equal(y.isnan(), ref.isnan())
            assert int(y.isnan().any(1).sum()) == (m > 6)
    assert ops.int8_status() == 0


@pytest.mark.parametrize("kernel", ["split", "pair"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m, n, k", [(1, 1000, 512), (19, 333, 700), (300, 520, 2050), (513, 1024, 640)])
def test_linear_forward(ops, m, n, k, dtype, kernel):
    x, w = _rand((m, k), dtype, 3), _rand((n, k), F32, 4, k ** -0.5)
    weights = ops.int8_quantize(w)
    ops.set_int8_kernel(kernel)
    try:
        for bias in (None, _rand((n,), F32, 5), _rand((n,), BF16, 5), _rand((n,), F16, 5)):
            ref, parts = _linear_ref(x, w, bias)
            y = ops.int8_linear(x, weights, bias)
            assert y.dtype == dtype and y.shape == (m, n)
            _check(y, ref, parts)
            assert torch.equal(y, ops.int8_linear(x, w, bias))            # weights quantised in the call
            assert torch.equal(y, ops.int8_linear(x, weights, bias))      # the same again
    finally:
        ops.set_int8_kernel("auto")
    assert ops.int8_status() == 0


def test_both_kernels_agree_and_rows_do_not_depend_on_the_batch(ops):
    x, weights = _rand((700, 900), BF16, 3), ops.int8_quantize(_rand((777, 900), F32, 4))
    ops.set_int8_kernel("pair")
    whole = ops.int8_linear(x, weights)
    ops.set_int8_kernel("split")
    assert torch.equal(whole, ops.int8_linear(x, weights))
    ops.set_int8_kernel("auto")
    for rows in (1, 2, 15, 16, 31, 64, 100, 128, 129, 400):
        assert torch.equal(ops.int8_linear(x[:rows], weights), whole[:rows])


def test_shapes_of_x(ops):
    w = _rand((50, 96), F32, 1)
    weights = ops.int8_quantize(w)
    x = _rand((2, 3, 4, 96), BF16, 2)
    y = ops.int8_linear(x, weights)
    assert y.shape == (2, 3, 4, 50)
    assert torch.equal(y[1, 2, 3], ops.int8_linear(x[1, 2, 3], weights))
    assert torch.equal(y.flatten(0, 2), ops.int8_linear(x.flatten(0, 2), weights))
    assert torch.equal(y.transpose(0, 2), ops.int8_linear(x.transpose(0, 2), weights))
    assert ops.int8_linear(x[:0], weights).shape == (0, 3, 4, 50)
    assert ops.int8_linear(x.double(), weights).dtype == F32
    assert torch.equal(ops.int8_linear(x, w.t().contiguous().t()), y)


def test_outputs_of_every_alignment(ops):
    # rows of the output that begin on 32, 16, 8, 4 or 2 bytes only
    x = _rand((270, 200), F32, 1)
    for n in (256, 264, 260, 258, 257, 1, 2, 31):
        w = _rand((n, 200), F32, n)
        for dtype in (F32, BF16):
            for kernel in ("split", "pair"):
                ops.set_int8_kernel(kernel)
                y = ops.int8_matmul(ops.int8_quantize(x), ops.int8_quantize(w), dtype=dtype)
                ops.set_int8_kernel("auto")
                _check(y, _linear_ref(x, w)[0])


def test_offsets_beyond_32_bits(ops):
    rows, cols = 40000, 65536
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    x[-3:] = _rand((3, cols), BF16, 1)
    x[0] = 1
    w = _rand((130, cols), BF16, 2)
    a, b = ops.int8_quantize(x), ops.int8_quantize(w)
    assert a.data.numel() > 2 ** 31
    for left, right in ((a, b), (b, a)):
        y = ops.int8_matmul(left, right)
        y = y if left is a else y.t()
        _check(y[-3:], _linear_ref(x[-3:], w)[0])
        _check(y[:1], _linear_ref(x[:1], w)[0])
        assert (y[1:-3] == 0).all()


# ---- gradients --------------------------------------------------------------------------------------------------
def _grads_ref(x, w, dy):
    """dx, dw, db by the definition, with what was added up for db."""
    (qx, sx), (qw, sw) = _quant(x), _quant(w)
    g = (dy.float() * sw.float()).double()
    h = (dy.float() * sx.float()[:, None]).double()
    (qg, sg), (qh, sh) = _quant(g), _quant(h, 0)
    return (qg @ qw) * sg[:, None], (qh.t() @ qx) * sh[:, None], dy.double().sum(0), dy.double().abs().sum(0)


@pytest.mark.parametrize("kernel", ["auto", "split", "pair"])
@pytest.mark.parametrize("xt, wt", [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("m, n, k", [(1, 5, 7), (2, 128, 128), (130, 1000, 512), (256, 300, 140), (515, 260, 1030)])
def test_gradients_are_those_of_the_definition(ops, m, n, k, xt, wt, kernel):
    x, w, b = _rand((m, k), xt, 1).requires_grad_(), _rand((n, k), wt, 2).requires_grad_(), _rand((n,), F32, 3).requires_grad_()
    dy = _rand((m, n), xt, 4, 1e-2)
    ops.set_int8_kernel(kernel)
    try:
        y = ops.int8_linear(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    finally:
        ops.set_int8_kernel("auto")
    assert ops.int8_status() == 0
    rx, rw, rb, parts = _grads_ref(x.detach(), w.detach(), dy)
    assert dx.dtype == xt and dw.dtype == wt and db.dtype == F32
    ry, rparts = _linear_ref(x.detach(), w.detach(), b.detach())
    _check(y.detach(), ry, rparts)
    _check(dx, rx)
    _check(dw, rw)
    # a sum of m numbers as 8 + 8 + m / 64 additions one behind the other
    assert ((db.double() - rb).abs() <= (16 + m / 64) * 2.0 ** -24 * parts).all()


def test_gradients_against_differences(ops):
    """The layer is linear in what its operands stand for, so differences of the exact products are what the gradients stand
    in for; a gradient is off by half a step of the quantised dy at every term."""
    m, n, k = 60, 70, 90
    x, w, dy = _rand((m, k), F32, 1), _rand((n, k), F32, 2), _rand((m, n), F32, 3)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ops.int8_linear(xr, wr), (xr, wr), dy)
    (qx, sx), (qw, sw) = _quant(x), _quant(w)
    xh, wh = qx * sx[:, None], qw * sw[:, None]
    loss = lambda a, b: (dy.double() * (a @ b.t())).sum()
    g, h = dy.double() * sw, dy.double() * sx[:, None]
    step_g, step_h = g.abs().amax(1) / 127, h.abs().amax(0) / 127
    for i, j in [(0, 0), (5, 17), (59, 89), (30, 44)]:
        d = torch.zeros_like(xh)
        d[i, j] = 0.5
        slope = loss(xh + d, wh) - loss(xh - d, wh)
        assert (dx[i, j].double() - slope).abs() <= 0.5001 * step_g[i] * qw[:, j].abs().sum() + 1e-9
        d = torch.zeros_like(wh)
        d[i, j] = 0.5
        slope = loss(xh, wh + d) - loss(xh, wh - d)
        assert (dw[i, j].double() - slope).abs() <= 0.5001 * step_h[i] * qx[:, j].abs().sum() + 1e-9


def test_which_gradients_are_computed(ops):
    x, w, b = _rand((20, 64)), _rand((30, 64), F32, 1), _rand((30,), F32, 2)
    dy = _rand((20, 30), F32, 3)
    full = None
    for mask in (7, 1, 2, 4, 3, 5, 6):
        args = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        y = ops.int8_linear(*args)
        y.backward(dy)
        got = [t.grad for t in args]
        full = full or got
        for i in range(3):
            assert (got[i] is not None) == bool(mask >> i & 1)
            assert got[i] is None or torch.equal(got[i], full[i])
    # prepared weights pass the gradient of x on
    xr = x.clone().requires_grad_()
    ops.int8_linear(xr, ops.int8_quantize(w), b).backward(dy)
    assert torch.equal(xr.grad, full[0])
    with torch.no_grad():
        assert not ops.int8_linear(xr, w, b).requires_grad


def test_gradients_of_broadcast_and_shared_tensors(ops):
    w = _rand((30, 64), F32, 1)
    row = _rand((1, 64), F32, 2)
    # one row broadcast to a batch: its gradient is the sum over the batch
    r1, r2 = row.clone().requires_grad_(), row.expand(12, 64).contiguous().requires_grad_()
    dy = _rand((12, 30), F32, 3)
    ops.int8_linear(r1.expand(12, 64), w).backward(dy)
    ops.int8_linear(r2, w).backward(dy)
    assert torch.allclose(r1.grad, r2.grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-6)
    # the same weight in two layers of a chain; dy with stride 0 (a sum)
    s = _rand((64, 64), F32, 4).requires_grad_()
    ops.int8_linear(ops.int8_linear(row.expand(12, 64), s), s).sum().backward()
    assert s.grad.isfinite().all() and s.grad.abs().sum() > 0
    # 3-dimensional x and a transposed weight view
    x3, wt = _rand((3, 5, 64), BF16, 5).requires_grad_(), w.t().contiguous().requires_grad_()
    d3 = _rand((3, 5, 30), BF16, 6)
    ops.int8_linear(x3, wt.t()).backward(d3)
    rx, rw, _, _ = _grads_ref(x3.detach().view(15, 64), w, d3.view(15, 30))
    _check(x3.grad.view(15, 64), rx)
    _check(wt.grad.t(), rw)


def test_types_beyond_the_kernels(ops):
    # float64 operands are computed as float32; their gradients come back in float64
    x, w = _rand((20, 64)).double().requires_grad_(), _rand((30, 64), F32, 1).double().requires_grad_()
    b = _rand((30,), F32, 2).double().requires_grad_()
    y = ops.int8_linear(x, w, b)
    dy = _rand((20, 30), F32, 3)
    y.backward(dy)
    assert y.dtype == F32 and x.grad.dtype == w.grad.dtype == b.grad.dtype == torch.float64
    rx, rw, _, _ = _grads_ref(x.detach().float(), w.detach().float(), dy)
    _check(x.grad.float(), rx)
    _check(w.grad.float(), rw)
    with torch.inference_mode():
        assert torch.equal(ops.int8_linear(x, w, b), y.detach())


def test_gradients_of_odd_batches(ops):
    w, b = _rand((30, 64), F32, 1).requires_grad_(), _rand((30,), F32, 1).requires_grad_()
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    ops.int8_linear(x, w, b).sum().backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all() and (b.grad == 0).all()
    # padded tokens: rows of zeros in x and in dy
    x = _rand((40, 64), F32, 2)
    x[::3] = 0
    dy = _rand((40, 30), F32, 3)
    dy[1::3] = 0
    xr = x.clone().requires_grad_()
    w.grad = b.grad = None
    ops.int8_linear(xr, w, b).backward(dy)
    rx, rw, rb, _ = _grads_ref(x, w.detach(), dy)
    _check(xr.grad, rx)
    _check(w.grad, rw)
    assert (xr.grad[1::3] == 0).all()
    # a token with a NaN: its own output and gradient, and the weights', are NaN; the other tokens' gradients are not
    x[5, 5] = float("nan")
    xr = x.clone().requires_grad_()
    w.grad = None
    y = ops.int8_linear(xr, w, b)
    y.backward(dy)
    assert y[5].isnan().all() and int(y.isnan().any(1).sum()) == 1
    assert w.grad.isnan().all() and xr.grad.isfinite().all()
    # an infinite gradient of one token: only its row of dx, its column of dw
    dy[7, 3] = float("inf")
    x[5, 5] = 0
    xr = x.clone().requires_grad_()
    w.grad = None
    ops.int8_linear(xr, w, b).backward(dy)
    assert xr.grad[7].isnan().all() and int(xr.grad.isnan().any(1).sum()) == 1
    assert w.grad[3].isnan().all() and int(w.grad.isnan().any(1).sum()) == 1


# ---- streams and graphs -----------------------------------------------------------------------------------------
def test_other_stream_and_two_streams_at_once(ops):
    x, w = _rand((300, 512), BF16, 1), _rand((640, 512), F32, 2)
    weights = ops.int8_quantize(w)
    ref = ops.int8_linear(x, weights)
    small = ops.int8_linear(x[:3], weights)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for turn in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append((i, ops.int8_linear(x if i else x[:3], weights)))
    torch.cuda.synchronize()
    for i, y in outs:
        assert torch.equal(y, ref if i else small)


def test_captured_forward_and_backward(ops):
    x, w = _rand((130, 256), BF16, 1).requires_grad_(), _rand((300, 256), F32, 2).requires_grad_()
    dy = _rand((130, 300), BF16, 3)

    def step():
        y = ops.int8_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    # (no eager graph of the same leaves may live through a capture: torch's engine would then wait on the stream of that
    #  graph's leaf nodes, which a capture does not allow, whatever the op)
    graphs = []
    for _ in range(2):                    # two graphs, each with its own scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for turn in range(3):
        with torch.no_grad():
            x.copy_(_rand((130, 256), BF16, 10 + turn))
            w.copy_(_rand((300, 256), F32, 20 + turn))
        ref = step()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, ref):
                assert torch.equal(a, b)


# ---- order of launches that begin under the end of the one before them --------------------------------------------
@pytest.mark.parametrize("m", [1, 8, 64, 600])
@pytest.mark.parametrize("kernel", ["auto", "split", "pair"])
def test_calls_behind_one_another(ops, m, kernel):
    """Weights quantised right before they are used, in memory that the call before still reads; tokens written right before
    by another kernel: the same as call by call."""
    n, k = 700, 1300
    xs, ws = [_rand((m, k), BF16, seed=i) for i in range(3)], [_rand((n, k), BF16, seed=10 + i, scale=0.1) for i in range(4)]
    ops.set_int8_kernel(kernel)
    try:
        want = {}
        for i in range(12):
            x = xs[i % 3] * 2
            torch.cuda.synchronize()
            w = ops.int8_quantize(ws[i % 4])
            torch.cuda.synchronize()
            want[i] = ops.int8_linear(x, w)
            torch.cuda.synchronize()
            del w
        got = []
        for i in range(120):
            x = xs[i % 3] * 2
            w = ops.int8_quantize(ws[i % 4])
            got.append(ops.int8_linear(x, w))
            del w, x
    finally:
        ops.set_int8_kernel("auto")
    assert all(torch.equal(y, want[i % 12]) for i, y in enumerate(got))
    assert ops.int8_status() == 0


@pytest.mark.parametrize("m, n, k", [(40, 256, 300), (600, 700, 500), (2000, 16, 2900)])
def test_training_steps_behind_one_another(ops, m, n, k):
    """Forward, backward and the step that changes the weights, without a pause and step by step."""
    from rexsc_b200 import optim

    xs, dys = [_rand((m, k), BF16, seed=i) for i in range(3)], [_rand((m, n), BF16, seed=5 + i) for i in range(3)]

    def train(pause):
        w, b = torch.nn.Parameter(_rand((n, k), F32, seed=9, scale=0.05)), torch.nn.Parameter(_rand((n,), seed=8))
        opt, out = optim.AdamW([w, b], lr=1e-2, state_bits=8), []
        for i in range(20):
            x = xs[i % 3].clone().requires_grad_()
            y = ops.int8_linear(x, w, b)
            pause()
            y.backward(dys[i % 3])
            pause()
            opt.step()
            pause()
            out += [y.detach(), x.grad, w.grad, b.grad]
            opt.zero_grad()
        return out + [w.detach(), b.detach()]

    for a, b in zip(train(lambda: None), train(torch.cuda.synchronize)):
        assert torch.equal(a, b)
    assert ops.int8_status() == 0


@pytest.mark.parametrize("before", ["nothing", "copy", "fill", "join"])
@pytest.mark.parametrize("m", [1, 64, 600])
def test_captured_behind_anything(ops, m, before):
    """What a call follows in a captured graph need not be a kernel."""
    x, w = _rand((m, 1300), BF16), ops.int8_quantize(_rand((700, 1300), BF16, seed=1))
    want, zero = ops.int8_linear(x, w), ops.int8_linear(torch.zeros_like(x), w)
    into, other = torch.zeros_like(x), torch.cuda.Stream()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    ops.int8_linear(into, w)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        if before == "copy":
            into.copy_(x)
        elif before == "fill":
            into.zero_()
        elif before == "join":
            other.wait_stream(stream)
            with torch.cuda.stream(other):
                into.copy_(x)
            into2 = into.new_ones(5) * 2
            stream.wait_stream(other)
        y = ops.int8_linear(into, w)
        z = ops.int8_linear(into, w)
    for fill in (x, torch.zeros_like(x)):
        into.copy_(fill)
        graph.replay()
        torch.cuda.synchronize()
        expect = want if before in ("copy", "join") or (before == "nothing" and fill is x) else zero
        assert torch.equal(y, expect) and torch.equal(z, expect)


# ---- refusals ---------------------------------------------------------------------------------------------------
def test_refusals(ops):
    x, w = _rand((4, 64)), _rand((8, 64))
    m = ops.int8_quantize(w)
    with pytest.raises(ValueError):
        ops.int8_linear(x[:, :63], m)
    with pytest.raises(ValueError):
        ops.int8_linear(x, w[0])
    with pytest.raises(ValueError):
        ops.int8_linear(x, m, _rand((9,)))
    with pytest.raises(ValueError):
        ops.int8_linear(x, m, torch.zeros(8))
    with pytest.raises(ValueError):
        ops.int8_linear(x.int(), m)
    with pytest.raises(ValueError):
        ops.int8_linear(x, w.to(torch.int8))
    with pytest.raises(RuntimeError):
        ops.int8_linear(x.cpu(), m)
    with pytest.raises(ValueError):
        ops.int8_quantize(x[:0])
    with pytest.raises(ValueError):
        ops.int8_quantize(x[0])
    with pytest.raises(ValueError):
        ops.int8_matmul(m, ops.int8_quantize(x[:, :32]))
    with pytest.raises(ValueError):
        ops.int8_matmul(m, m, dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.int8_matmul(x, m)
    with pytest.raises(ValueError):
        ops.Int8Matrix.from_values(x, torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        ops.Int8Matrix.from_values(m.values(), torch.ones(4, device="cuda"))
    long = ops.int8_quantize(torch.ones(2, 131072, device="cuda"))
    with pytest.raises(ValueError):
        ops.int8_matmul(long, long)
    with pytest.raises(ValueError):
        ops.int8_linear(torch.ones(2, 131072, device="cuda"), long)
    most = ops.int8_quantize(torch.ones(2, 131071, device="cuda"))
    assert (ops.int8_matmul(most, most) - 131071).abs().max() <= 131071 * 4 * 2.0 ** -24
    with pytest.raises(ValueError):
        ops.int8_linear(torch.ones(131072, 8, device="cuda"), torch.ones(4, 8, device="cuda", requires_grad=True))
    y = ops.int8_linear(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError):   # no second derivative
        g, = torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)
        g.sum().backward()


def test_matrices_that_do_not_fit_their_size_are_refused(ops):
    """Nothing is launched: each is refused when it is made, or by the check of the call."""
    m = ops.int8_quantize(_rand((200, 300)))
    for rows, cols, data, scale in [(200, 300, m.data[:-1], m.scale), (200, 400, m.data, m.scale), (0, 300, m.data, m.scale),
                                    (200, 300, m.data.float(), m.scale), (200, 300, m.data, m.scale[:-1]),
                                    (200, 300, m.data, m.scale.double()), (200, 300, m.data, m.scale.cpu()),
                                    (200, 300, torch.cat([m.data, m.data])[16:16 + m.data.numel()], m.scale),
                                    (200, 300, m.data, torch.stack([m.scale, m.scale], 1)[:, 0])]:
        with pytest.raises(ValueError):
            ops.Int8Matrix(rows, cols, data, scale)
    with pytest.raises(RuntimeError):
        ops.Int8Matrix(200, 300, m.data.cpu(), m.scale)
    for name in ("rows", "cols", "data", "scale"):
        with pytest.raises(AttributeError):
            setattr(m, name, getattr(m, name))
    gone = ops.int8_quantize(_rand((200, 300)))
    gone.data.resize_(16)
    with pytest.raises(ValueError):
        ops.int8_linear(_rand((4, 300)), gone)
    with pytest.raises(ValueError):
        ops.int8_matmul(gone, gone)
    with pytest.raises(ValueError):
        gone.values()


def test_copies_of_a_matrix(ops):
    import copy
    import pickle

    m, x = ops.int8_quantize(_rand((200, 300))), _rand((5, 300), seed=1)
    y = ops.int8_linear(x, m)
    for other in (copy.deepcopy(m), copy.copy(m), pickle.loads(pickle.dumps(m)), ops.Int8Matrix(200, 300, m.data.clone(), m.scale.clone())):
        assert other.shape == (200, 300) and torch.equal(ops.int8_linear(x, other), y)
