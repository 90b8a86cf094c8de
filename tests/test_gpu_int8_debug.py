"""REXSC_B200_DEBUG=1: a product whose waits gave up raises by itself, in each call that has one."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import torch
from rexsc_b200 import _lib, ops

lib = _lib.load()
g = torch.Generator(device="cuda").manual_seed(0)
x = torch.randn(60, 300, generator=g, device="cuda", requires_grad=True)
w = torch.randn(200, 300, generator=g, device="cuda", requires_grad=True)
w8 = ops.int8_quantize(w)


def raises(call):
    lib.rexsc_int8_test_waits(-2)
    try:
        call()
    except RuntimeError as e:
        return "REXSC_E_DEVICE_TIMEOUT" in str(e)
    finally:
        lib.rexsc_int8_test_waits(-1)
        ops.int8_status()
    return False


y = ops.int8_linear(x, w)
print("serving", raises(lambda: ops.int8_linear(x.detach(), w8)))
print("one token", raises(lambda: ops.int8_linear(x.detach()[0], w8)))
print("training", raises(lambda: ops.int8_linear(x, w)))
print("matmul", raises(lambda: ops.int8_matmul(w8, w8)))
print("backward", raises(lambda: y.sum().backward()))

ref, inputs = ops.int8_linear(x.detach(), w8), x.detach()
both = ops.int8_matmul(w8, w8)
graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
leaves = [t.detach().clone().requires_grad_() for t in (x, w)]
grads = torch.autograd.grad(ops.int8_linear(*leaves).sum(), leaves)
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=stream):
    y, z = ops.int8_linear(inputs, w8), ops.int8_matmul(w8, w8)
    again = torch.autograd.grad(ops.int8_linear(*leaves).sum(), leaves)
graph.replay()
torch.cuda.synchronize()
print("captured", torch.equal(y, ref) and torch.equal(z, both) and all(torch.equal(a, b) for a, b in zip(grads, again)))
"""


@pytest.mark.parametrize("debug", ["1", "0"])
def test_status_of_every_product(ops, debug):
    env = {**os.environ, "REXSC_B200_DEBUG": debug, "PYTHONPATH": ROOT}
    run = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=180, env=env, cwd=ROOT)
    assert run.returncode == 0, run.stderr[-2000:]
    said = dict(line.rsplit(" ", 1) for line in run.stdout.strip().splitlines())
    assert said.pop("captured") == "True"
    assert said == dict.fromkeys(["serving", "one token", "training", "matmul", "backward"], str(debug == "1"))
