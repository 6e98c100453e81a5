"""The norms of the block glue on tensors that start off 16-byte borders (slices of a flat buffer of parameters, say): the C
entry points refuse them, the Python ones copy."""
import ctypes

import pytest
import torch

import verace_v1_b200 as V
from verace_v1_b200 import _lib


@pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers: run without a GPU only")
def test_entry_points_refuse_unaligned_pointers():
    L = _lib.lib()
    good, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)
    for i in range(3):
        p = [good] * 3
        p[i] = odd
        assert L.verace_rmsnorm(*p, 2, 64, 1e-6, 1, None) == 1 and b"aligned" in L.verace_last_error()
    for i in range(5):
        p = [good] * 5
        p[i] = odd
        h, y, wy, wn, n = p
        assert L.verace_add_rmsnorm(h, y, 1, wy, 1e-6, wn, 1e-6, n, 2, 64, 1, None) == 1 and b"aligned" in L.verace_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [64, 128, 1024, 2048])
def test_tensors_off_their_borders(dt, cols):
    g = torch.Generator(device="cuda").manual_seed(cols)

    def made(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)

    def moved(t):
        flat = torch.zeros(t.numel() + 8, device="cuda", dtype=dt)
        flat[1:1 + t.numel()] = t.reshape(-1)
        return flat[1:1 + t.numel()].view(t.shape)
    x, y, w, u = made(5, cols), made(5, cols), made(cols), made(cols)
    a, b = (torch.nn.RMSNorm(cols, device="cuda", dtype=dt).requires_grad_(False) for _ in range(2))
    c, d = (torch.nn.RMSNorm(cols, device="cuda", dtype=dt) for _ in range(2))
    a.weight.copy_(w), b.weight.copy_(u)
    c.weight, d.weight = torch.nn.Parameter(moved(w)), torch.nn.Parameter(moved(u))
    assert c.weight.data_ptr() % 16
    want = V.rmsnorm(x, a)
    assert torch.equal(V.rmsnorm(moved(x), a), want) and torch.equal(V.rmsnorm(x, c), want)
    h0, h1, h2 = x.clone(), moved(x), x.clone()
    n0 = V.add_rmsnorm(h0, y, a, b)
    version = h1._version
    n1, n2 = V.add_rmsnorm(h1, moved(y), c, d), V.add_rmsnorm(h2, moved(y), c, b)
    assert torch.equal(n0, n1) and torch.equal(n0, n2) and torch.equal(h0, h1) and torch.equal(h0, h2) and h1._version > version
