"""The bias's gradient of int8_linear: the error of the sum does not grow with the number of tokens.

A warp of the first pass adds up one row in eight of a block one by one in fp32: 32 rows of blocks of 256, as they are up to
32768 tokens, at most 31 half steps of what was added up.  A block's sum is rounded once and the result once: 33 in all.  What a
large value leaves no room for in its own warp is lost, and no more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _bias_gradient(ops, dy, btype=F32, all_three=True):
    m, n = dy.shape
    x = torch.ones(m, 8, device="cuda", dtype=dy.dtype, requires_grad=all_three)
    w = torch.ones(n, 8, device="cuda", requires_grad=all_three)
    b = torch.zeros(n, device="cuda", dtype=btype, requires_grad=True)
    return torch.autograd.grad(ops.int8_linear(x, w, b), b, dy)[0]


@pytest.mark.parametrize("all_three", [True, False])
@pytest.mark.parametrize("m, n", [(256, 1000), (1000, 70), (8192, 300), (32768, 5)])
def test_many_small_values_beside_a_large_one(ops, m, n, all_three):
    """One 1 and else 2^-31: each warp's sum is below half a step of 1, all of them together are many steps (from 8192 tokens
    on).  Exact but for the large value's warp (31 lost values of 2^-31), its block's rounding and the result's."""
    dy = torch.full((m, n), 2.0 ** -31, device="cuda")
    rows = (torch.arange(n, device="cuda") * 37) % m
    dy[rows, torch.arange(n, device="cuda")] = 1.0
    got = _bias_gradient(ops, dy, all_three=all_three)
    ref = dy.double().sum(0)
    assert ((got.double() - ref).abs() <= 31 * 2.0 ** -31 + 2 * 2.0 ** -24 * ref).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("btype", [F32, F16, BF16])
@pytest.mark.parametrize("m, n", [(1, 9), (257, 130), (3001, 257), (30000, 33)])
def test_sums(ops, m, n, dtype, btype):
    dy = torch.randn(m, n, generator=torch.Generator(device="cuda").manual_seed(m), device="cuda").to(dtype)
    got = _bias_gradient(ops, dy, btype)
    assert got.dtype == btype
    ref, parts = dy.double().sum(0), dy.double().abs().sum(0)
    allowed = 32 * 2.0 ** -24 * parts
    allowed = allowed + (ref.abs() + allowed) * torch.finfo(btype).eps / 2 + torch.finfo(btype).smallest_normal * torch.finfo(btype).eps / 2
    assert ((got.double() - ref).abs() <= allowed).all()


def test_special_values(ops):
    dy = torch.ones(600, 6, device="cuda")
    dy[300, 0], dy[10, 1], dy[500, 2] = float("inf"), float("nan"), -float("inf")
    dy[5, 2] = float("inf")
    dy[:, 3] = 3e38
    got = _bias_gradient(ops, dy)
    assert got[0] == float("inf") and got[1].isnan() and got[2].isnan() and got[3] == float("inf")
    assert (got[4:] == 600).all()
    for dtype in (F16, BF16):
        got = _bias_gradient(ops, dy, dtype)
        assert got[0] == float("inf") and got[1].isnan() and got[3] == float("inf")
