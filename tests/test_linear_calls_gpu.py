"""The dense products and the 8-bit norm in the places a program calls them from: threads, orders of calls, tensors
that other calls write."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import verace_v1_b200 as V
from linear_util import assert_within, linear64

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HERE = os.path.dirname(os.path.abspath(__file__))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def test_first_call_of_a_thread():
    """A thread whose first call of CUDA is a product (its memory comes out of the cache)."""
    g = gen(1)
    x, w, big = randn(g, 64, 256, dt=BF16), randn(g, 512, 256, dt=BF16), randn(g, 300, 256, dt=BF16)
    q4, s4, _ = V.quantize_int4(w)
    calls = [lambda: V.fused_linear(x, w), lambda: V.fused_linear(big, w), lambda: V.gated_linear(x, w, w),
             lambda: V.int4_linear(x[:8], q4, s4)]
    want = [c() for c in calls]
    for i in range(len(calls)):
        got = []

        def work():
            try:
                got.append(calls[i]())
            except Exception as e:      # (a thread's own errors reach nobody)
                got.append(e)
        calls[i]()
        torch.cuda.synchronize()
        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert isinstance(got[0], torch.Tensor), got[0]
        assert torch.equal(got[0], want[i])


FIRST = """
import conftest, torch
import verace_v1_b200 as V
g = torch.Generator(device="cuda").manual_seed(2)
x, w, d = (torch.randn(*s, device="cuda", generator=g).bfloat16() for s in ((300, 128), (256, 128), (300, 256)))
torch.cuda.synchronize()
x.requires_grad_(%s), w.requires_grad_()
y = V.fused_linear(x, w)
spare = [torch.empty(1 << 22, device="cuda") for _ in range(4)]     # (what the backward asks for is in the cache)
del spare
y.backward(d)
want = d.double().t() @ x.double()
assert ((w.grad.double() - want).norm() / want.norm()) < 4e-3
print("done")
"""


@pytest.mark.parametrize("wants", [False, True])
def test_first_backward_of_a_process(wants):
    """Autograd's own thread, whose first call is a product of operands as they lie (no bias, no activation)."""
    r = subprocess.run([sys.executable, "-c", FIRST % wants], cwd=HERE, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr
