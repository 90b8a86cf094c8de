"""Arguments of the int8 and AdamW entry points, checked without a GPU: nothing is launched."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from rexsc_b200 import _lib, build

    build.build()
    return _lib.load()


def test_sizes_of_8_bit_matrices(lib):
    tile = 128 * 128
    for rows, cols, tiles in [(1, 1, 1), (128, 128, 1), (129, 128, 2), (128, 129, 2), (1000, 512, 32), (1 << 20, 1 << 16, 1 << 22)]:
        assert lib.rexsc_int8_data_size(rows, cols) == tiles * tile
    for rows, cols in [(0, 1), (1, 0), (-1, 5), ((1 << 30) + 1, 1)]:
        assert lib.rexsc_int8_data_size(rows, cols) == 0
    assert lib.rexsc_int8_linear_workspace_size(17, 4096, 4096, 0) == 256 + 32 * tile
    assert lib.rexsc_int8_linear_workspace_size(4, 4096, 4096, 0) == 0           # the product's kernel quantises a few tokens
    assert lib.rexsc_int8_linear_workspace_size(16, 512, 512, 0) == 0
    assert lib.rexsc_int8_linear_workspace_size(16, 4096, 4096, 2) == 256 + 32 * tile
    assert lib.rexsc_int8_linear_workspace_size(1, 8, 131071, 0) == 256 + 1024 * tile   # too long for that
    assert lib.rexsc_int8_linear_workspace_size(17, 4096, 131072, 0) == 0
    both = lib.rexsc_int8_linear_bwd_workspace_size(300, 500, 1, 1, 1)
    assert both > 2 * 3 * 4 * tile
    assert lib.rexsc_int8_linear_bwd_workspace_size(300, 500, 1, 0, 0) < both
    assert lib.rexsc_int8_linear_bwd_workspace_size(0, 500, 1, 1, 1) == 0


def test_int8_entry_points_refuse_bad_arguments(lib):
    p = C.c_void_p(4096)
    off = C.c_void_p(4096 + 16)
    q = lib.rexsc_int8_quantize
    assert q(None, 0, 4, 4, 4, p, p, None) == -1
    assert q(p, 3, 4, 4, 4, p, p, None) == -1
    assert q(p, 0, 0, 4, 4, p, p, None) == -1
    assert q(p, 0, 4, 4, -1, p, p, None) == -1
    assert q(p, 0, 4, 4, 4, off, p, None) == -1
    assert lib.rexsc_int8_pack(p, 4, 4, 4, None, None) == -1
    assert lib.rexsc_int8_unpack(p, 4, 0, p, None) == -1
    mm = lib.rexsc_int8_matmul
    assert mm(p, p, p, p, None, 0, 4, 4, 131072, p, 0, 0, None) == -4
    assert mm(p, p, p, p, None, 0, 4, 4, 128, p, 0, 3, None) == -1
    assert mm(p, p, p, p, p, 9, 4, 4, 128, p, 0, 0, None) == -1
    assert mm(p, None, p, p, None, 0, 4, 4, 128, p, 0, 0, None) == -1
    assert mm(off, p, p, p, None, 0, 4, 4, 128, p, 0, 0, None) == -1
    fwd = lib.rexsc_int8_linear_fwd
    assert fwd(p, 0, 400, 128, 128, p, p, 8, None, 0, p, 0, 0, None, 0, None) == -3
    assert fwd(p, 0, 400, 128, 128, p, p, 8, None, 0, p, 0, 0, p, 256, None) == -3
    assert fwd(p, 0, 400, 128, 128, off, p, 8, None, 0, p, 0, 0, p, 1 << 30, None) == -1
    train = lib.rexsc_int8_linear_train_fwd
    assert train(p, 0, 4, 128, 128, p, 0, 8, 128, None, 0, off, p, p, p, p, 0, 0, None) == -1
    assert train(p, 0, 4, 128, 128, p, 7, 8, 128, None, 0, p, p, p, p, p, 0, 0, None) == -1
    assert train(p, 0, 4, 128, 128, p, 0, 8, 128, None, 0, p, None, p, p, p, 0, 0, None) == -1
    assert train(p, 0, 4, 131072, 131072, p, 0, 8, 131072, None, 0, p, p, p, p, p, 0, 0, None) == -4
    assert fwd(p, 0, 4, 131072, 131072, p, p, 8, None, 0, p, 0, 0, p, 1 << 40, None) == -4
    bwd = lib.rexsc_int8_linear_bwd
    assert bwd(p, 0, 4, 8, 128, 8, p, p, p, p, None, 0, None, 0, None, 0, 0, p, 1 << 30, None) == -1   # nothing wanted
    assert bwd(p, 0, 4, 8, 128, 8, p, p, None, None, p, 0, None, 0, None, 0, 0, p, 1 << 30, None) == -1  # dx without w
    assert bwd(p, 0, 4, 131072, 128, 8, p, p, p, p, p, 0, None, 0, None, 0, 0, p, 1 << 40, None) == -4
    assert bwd(p, 0, 4, 8, 128, 8, p, p, p, p, p, 0, p, 0, p, 0, 0, p, 16, None) == -3


def _adamw(**kw):
    from rexsc_b200 import _lib

    d = _lib.AdamWDesc()
    base = dict(state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, d_step=4096, d_exp_avg=4096,
                d_exp_avg_sq=4096)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def test_adamw_entry_point_refuses_bad_arguments(lib):
    from rexsc_b200 import _lib

    def call(tensors=((4096, 4096, 10, 0),), **kw):
        d = _adamw(**kw)
        t = (_lib.AdamWTensor * max(1, len(tensors)))(*[_lib.AdamWTensor(*v) for v in tensors])
        return lib.rexsc_adamw_step(C.byref(d), C.addressof(t), len(tensors), None)

    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1e-8),
                dict(weight_decay=-1.0), dict(param_dtype=3), dict(grad_dtype=-1), dict(d_step=None), dict(d_exp_avg=None),
                dict(d_exp_avg=4096 + 16), dict(state_bits=8)):
        assert call(**bad) == -1, bad
    assert call(tensors=((None, 4096, 10, 0),)) == -1
    assert call(tensors=((4096, None, 10, 0),)) == -1
    assert call(tensors=((4096, 4096, 0, 0),)) == -1
    assert call(tensors=((4096, 4096, 257, 0), (4096, 4096, 10, 1))) == -1     # overlap
    assert call(tensors=((4096, 4096, 10, 1 << 31),)) == -4
    assert lib.rexsc_adamw_step(None, None, 0, None) == -1
    assert call(tensors=()) == 0                                              # nothing to do


def test_python_side_refuses_cpu_tensors():
    from rexsc_b200 import ops, optim

    with pytest.raises(RuntimeError):
        ops.int8_quantize(torch.zeros(4, 4))
    with pytest.raises(RuntimeError):
        ops.int8_linear(torch.zeros(4, 4), torch.zeros(4, 4))
    with pytest.raises(RuntimeError):
        ops.Int8Matrix.from_values(torch.zeros(4, 4, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(ValueError):
        ops.int8_matmul(torch.zeros(4, 4), torch.zeros(4, 4))
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(), dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
