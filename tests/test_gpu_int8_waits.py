"""What an int8 product does when a bounded wait gives up: the status says so, and nothing that was not computed is stored.

The library makes the waits of chosen blocks give up at once; copies and products in flight are still waited for, so nothing is
left running and the next call works."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
OUT = 0.5           # what the outputs hold before a call (no sum of integers)


@pytest.fixture()
def lib(ops):
    from rexsc_b200 import _lib

    lib = _lib.load()
    yield lib
    lib.rexsc_int8_test_waits(-1)
    ops.int8_status()


def _ints(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, (rows, cols), generator=g, device="cuda").to(torch.int8)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _matmul(lib, ops, a, b, kernel):
    out = torch.full((a.rows, b.rows), OUT, device="cuda")
    rc = lib.rexsc_int8_matmul(a.data.data_ptr(), a.scale.data_ptr(), b.data.data_ptr(), b.scale.data_ptr(), None, 0, a.rows, b.rows,
                               a.cols, out.data_ptr(), 0, kernel, _stream())
    assert rc == 0
    return out


# contractions of one step, of as many as a ring of stages holds, and of many more; clusters of 1, 2, 4 and 8
@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("m, n, k", [(5, 130, 100), (16, 128, 1024), (40, 300, 4096), (128, 512, 520), (300, 3000, 700),
                                     (260, 260, 20000), (2600, 2700, 300)])
def test_waits_that_give_up_store_nothing(lib, ops, m, n, k, kernel):
    qa, qb = _ints(m, k, 1), _ints(n, k, 2)
    a, b = (ops.Int8Matrix.from_values(q, torch.ones(len(q), device="cuda")) for q in (qa, qb))
    ref = (qa.double() @ qb.double().t()).float()
    assert lib.rexsc_int8_test_waits(-2) == 0
    out = _matmul(lib, ops, a, b, kernel)
    assert ops.int8_status() == -6 and ops.int8_status() == 0
    assert (out == OUT).all()
    if kernel == 1:     # one block: what its cluster would have joined, and nothing else
        rows = 128 if m > 64 else 64 if m > 32 else 32 if m > 16 else 16
        for block in (0, 1):
            assert lib.rexsc_int8_test_waits(block) == 0
            out = _matmul(lib, ops, a, b, kernel)
            assert ops.int8_status() == -6
            lost = out == OUT
            assert torch.equal(out[~lost], ref[~lost])
            tiles = {(i // rows, j // 128) for i, j in lost.nonzero()[:: 97].tolist()}
            assert len(tiles) == 1
            i, j = tiles.pop()
            assert lost[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128].all()
            assert int(lost.sum()) == lost[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128].numel()
    lib.rexsc_int8_test_waits(-1)
    assert torch.equal(_matmul(lib, ops, a, b, kernel), ref)
    assert ops.int8_status() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m, n, k", [(1, 300, 4096), (1, 2000, 128), (4, 4096, 1000), (16, 500, 700)])
def test_a_few_tokens(lib, ops, m, n, k, dtype):
    from rexsc_b200 import _lib

    x = torch.randn(m, k, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    w = ops.int8_quantize(torch.randn(n, k, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda"))
    assert lib.rexsc_int8_linear_workspace_size(m, n, k, 0) == 0        # the product's kernel quantises them
    code = {F32: _lib.F32, F16: _lib.F16, BF16: _lib.BF16}[dtype]

    def call():
        out = torch.full((m, n), OUT, device="cuda", dtype=dtype)
        assert lib.rexsc_int8_linear_fwd(x.data_ptr(), code, m, k, k, w.data.data_ptr(), w.scale.data_ptr(), n, None, 0,
                                         out.data_ptr(), code, 0, None, 0, _stream()) == 0
        return out

    ref = ops.int8_linear(x, w)
    lib.rexsc_int8_test_waits(-2)
    assert (call() == OUT).all()
    assert ops.int8_status() == -6
    lib.rexsc_int8_test_waits(0)
    out = call()
    assert ops.int8_status() == -6
    assert (out[:, :128] == OUT).all() and torch.equal(out[:, 128:], ref[:, 128:])
    lib.rexsc_int8_test_waits(-1)
    assert torch.equal(call(), ref)
    assert ops.int8_status() == 0


@pytest.mark.parametrize("kernel", ["split", "pair"])
def test_both_gradients(lib, ops, kernel):
    """Two products in one launch, or in two: neither hangs, and the calls that follow are right."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(200, 300, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(400, 300, generator=g, device="cuda", requires_grad=True)
    dy = torch.randn(200, 400, generator=g, device="cuda")
    ops.set_int8_kernel(kernel)
    try:
        ref = torch.autograd.grad(ops.int8_linear(x, w), (x, w), dy)
        y = ops.int8_linear(x, w)
        lib.rexsc_int8_test_waits(-2)
        torch.autograd.grad(y, (x, w), dy)
        assert ops.int8_status() == -6
        lib.rexsc_int8_test_waits(-1)
        got = torch.autograd.grad(ops.int8_linear(x, w), (x, w), dy)
    finally:
        ops.set_int8_kernel("auto")
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert ops.int8_status() == 0
