"""Values of eps that fp32 does not hold as a normal number are refused; checked without a GPU, nothing is launched."""
import ctypes as C

import pytest
import torch


def test_entry_point():
    from rexsc_b200 import _lib, build

    build.build()
    lib = _lib.load()

    def call(eps):
        d = _lib.AdamWDesc()
        for k, v in dict(state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=eps, d_step=4096, d_exp_avg=4096, d_exp_avg_sq=4096).items():
            setattr(d, k, v)
        return lib.rexsc_adamw_step(C.byref(d), None, 0, None)       # no tensors: nothing to do

    for eps in (0.0, 2.0 ** -126, 1e-30, 1e-8, 1.0, 1e30):
        assert call(eps) == 0, eps
    for eps in (1e-40, 2.0 ** -127, 5e-324, 1e-50, 1e38, float("inf"), float("nan"), -1e-8):
        assert call(eps) == -1, eps


@pytest.mark.parametrize("eps", [1e-40, 1e-50, 1e38, float("inf")])
def test_optimizer(eps):
    from rexsc_b200 import optim

    with pytest.raises(ValueError, match="normal number"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4))], eps=eps)
