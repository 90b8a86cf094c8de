"""Gradients of int8_linear where a block of the first pass takes several tiles of columns (more than 4096 output channels) or
more than 256 rows (more than 32768 tokens), against their definition.

dx and dw: exact sums of products, so the roundings of ``test_gpu_int8``.  db: a warp adds up at most 40 rows one by one, each a
rounding of the magnitudes added up so far, and two roundings follow: 41 half steps."""
import pytest
import torch

from test_gpu_int8 import BF16, F16, F32, _check, _grads_ref, _rand

pytestmark = pytest.mark.gpu

# tiles of a block / blocks: 2 / 10 (the last has one), 2 / 10, 2 / 16, 3 / 12; rows of a block: 264, 320
SIZES = [(130, 4700, 40), (64, 5003, 33), (300, 8192, 24), (17, 9000, 20), (33000, 300, 9), (40000, 70, 30), (1, 5003, 7)]


def _gradients(ops, x, w, dy):
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_(), torch.zeros(w.shape[0], device="cuda", requires_grad=True)]
    return torch.autograd.grad(ops.int8_linear(*leaves), leaves, dy)


def _same_rows(got, ref):
    """Rows that are NaN are the definition's; the others agree."""
    bad = ref.isnan().any(1)
    assert torch.equal(got.isnan().any(1), bad) and got[bad].isnan().all()
    _check(got[~bad], ref[~bad])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_against_the_definition(ops, m, n, k, dtype):
    x, w, dy = _rand((m, k), dtype, 1), _rand((n, k), F32, 2), _rand((m, n), dtype, 3, 1e-2)
    # the largest magnitude of a row in its first, second or last tile of a block, of a column in every part of the rows
    at = torch.arange(m, device="cuda")
    dy[at, (at * 131) % n] *= 50
    dy[at, n - 1 - (at * 7) % min(n, 300)] *= 20
    dx, dw, db = _gradients(ops, x, w, dy)
    rx, rw, rb, parts = _grads_ref(x, w, dy)
    _check(dx, rx)
    _check(dw, rw)
    assert ((db.double() - rb).abs() <= 41 * 2.0 ** -24 * parts).all()
    # without one or the other
    for want in ((0,), (1,), (0, 2), (1, 2), (2,)):
        leaves = [t.clone().requires_grad_(i in want) for i, t in enumerate((x, w, torch.zeros(n, device="cuda")))]
        got = torch.autograd.grad(ops.int8_linear(*leaves), [leaves[i] for i in want], dy)
        assert all(torch.equal(g, (dx, dw, db)[i]) for i, g in zip(want, got))
    assert ops.int8_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("m, n, k", [(130, 4700, 40), (64, 9000, 33), (40000, 70, 30)])
def test_what_is_no_number(ops, m, n, k, value, dtype):
    x, w, dy = _rand((m, k), dtype, 1), _rand((n, k), F32, 2), _rand((m, n), dtype, 3, 1e-2)
    places = [(0, n - 1), (m - 1, 300 % n), (m // 2, n // 2), (m // 3, (n // 3) | 1)]
    for i, j in places:
        dy[i, j] = value
    dx, dw, db = _gradients(ops, x, w, dy)
    rx, rw, _, _ = _grads_ref(x, w, dy)
    assert int(rx.isnan().any(1).sum()) == 4 and int(rw.isnan().any(1).sum()) == 4
    _same_rows(dx, rx)
    _same_rows(dw, rw)
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[[j for _, j in places]] = False
    assert db[fine].isfinite().all() and not db[~fine].isfinite().any()
