"""How near the dense products come: fp32 operands over fp32's whole range, errors in the 2-norm that the elementwise
bounds of linear_util.py would let pass, and sums that have to come out exactly.

Tolerances, derived before any run.  A dense product of fp32 operands keeps 24 bits of each operand (the pairs of parts that
are left out are below 2^-26 of a product).  64 values at a time are summed in the tensor core, where each of the last four
steps cuts at most 2^-23, 0.35 2^-23 on average, of what it has; the K / 64 sums are then added with rounding (0.2 2^-23 rms of
the running sum, which grows with the root of its length).  For random signs that is sqrt(4^2 0.35^2 + 0.2^2 K / 128) 2^-23 of
the result's 2-norm: 1.7e-7, and 3.4e-7 at K = 20000.  1e-6 is held; operands of two parts instead of three are
2e-6 off at best (2^-18 / sqrt(3) a value, both operands).  The engine of dot products is nearer.

16- and 8-bit operands are summed in the tensor core over all of K, 16 (8 bits: 32) values a step: K / 16 steps, each cutting at
most 2^-23 of a running sum of sqrt(i / K) of the result, together (2/3) K / 16 2^-23.
"""
import math

import pytest
import torch

import verace_v1_b200 as V
from linear_util import F64, act64, dequantised, fp8_rows

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MOST = torch.finfo(F32).max


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def off(got, want):
    """The error's 2-norm over the result's."""
    return float((got.to(F64) - want).norm() / want.norm())


# ---------------------------------------------------------------------------- fp32 operands of any size
def any_size(g, *shape):
    """Values whose exponents are spread over all of fp32's normal numbers, with the ends among them."""
    t = torch.randn(*shape, device="cuda", generator=g, dtype=F64)
    t = t.sign() * (1 + torch.rand(*shape, device="cuda", generator=g, dtype=F64))
    t = torch.ldexp(t, torch.randint(-126, 127, shape, device="cuda", generator=g).to(F64)).to(F32)
    ends = torch.tensor([MOST, -MOST, 2.0 ** -126, -(2.0 ** -126), 3.3895314e38, 3.3961775e38, -3.4e38, 1e-34, 1.2e-37, 1e-36],
                        device="cuda")
    t.view(-1)[:ends.numel()] = ends
    return t


@pytest.mark.parametrize("m,k", [(5, 64), (26, 100), (300, 130)])
def test_parts_of_every_size(m, k):
    """One weight of 1 a row: a value of x comes out, of whatever size, to the last step of the sum (2^-23 of it).  The
    same with x and the weights in each other's place, and in the gradients."""
    g = gen(m)
    x = any_size(g, m, k)
    n = 96
    pick = torch.randint(0, k, (n,), device="cuda", generator=g)
    pick[:10] = torch.arange(10, device="cuda")
    w = torch.zeros(n, k, device="cuda")
    w[torch.arange(n, device="cuda"), pick] = 1.0

    def close(got, want):
        assert bool(((got.to(F64) - want.to(F64)).abs() <= 2.0 ** -23 * want.to(F64).abs()).all()), off(got, want.to(F64))
    close(V.fused_linear(x, w), x[:, pick])
    close(V.fused_linear(w, x), x[:, pick].t())
    close(V.gated_linear(w, x, torch.ones_like(x), activation="relu"), torch.relu(x[:, pick].t()))     # (up: 1)
    # gradients: d picks rows and columns
    d, a = any_size(g, m, n), torch.zeros(m, k, device="cuda").requires_grad_()
    b = w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(V.fused_linear(a, b), (a, b), d)
    single = torch.zeros(n, k, device="cuda")
    single[torch.arange(min(n, k), device="cuda"), torch.arange(min(n, k), device="cuda")] = 1.0
    c = single.clone().requires_grad_()
    dx = torch.autograd.grad(V.fused_linear(a, c), a, d)[0]
    close(dx[:, :min(n, k)], d[:, :min(n, k)])
    rows = torch.zeros(m, k, device="cuda")
    rows[torch.arange(min(m, k), device="cuda"), torch.arange(min(m, k), device="cuda")] = 1.0
    dw = torch.autograd.grad(V.fused_linear(rows, c), c, d)[0]
    close(dw[:, :min(m, k)], d[:min(m, k)].t())


@pytest.mark.parametrize("scale", [1e-36, 1e-34, 1e-30, 1.0, 1e30, 1e36])
def test_sums_of_small_and_large_values(scale):
    g = gen(1)
    x, w = randn(g, 300, 500) * scale, randn(g, 130, 500) / 32
    want = x.to(F64) @ w.to(F64).t()
    assert off(V.fused_linear(x, w), want) < 1e-6
    assert off(V.fused_linear(w, x), want.t()) < 1e-6
    a, b = x.requires_grad_(), w.requires_grad_()
    d = randn(g, 300, 130) * 2.0 ** -6
    dx, dw = torch.autograd.grad(V.fused_linear(a, b), (a, b), d)
    assert off(dw, d.to(F64).t() @ x.to(F64)) < 1e-6 and off(dx, d.to(F64) @ w.to(F64)) < 1e-6


def test_an_infinity_in_fp32():
    """Up to 24 rows (gated: 16) what the formula gives; of more rows NaN, in the outputs that it enters and nowhere else."""
    g = gen(2)
    w = randn(g, 96, 64)
    for m in (4, 24, 25, 260):
        x = randn(g, m, 64)
        clean, gate = V.fused_linear(x, w), V.gated_linear(x, w, w)
        x[2, 7], x[3, 9] = math.inf, -math.inf
        y, h = V.fused_linear(x, w), V.gated_linear(x, w, w, activation="silu")
        keep = [i for i in range(m) if i not in (2, 3)]
        assert torch.equal(y[keep], clean[keep])
        if m <= 24:
            assert torch.equal(y[2], math.inf * w[:, 7].sign()) and torch.equal(y[3], -math.inf * w[:, 9].sign())
        else:
            assert y[2:4].isnan().all()
        if m > 16:
            assert h[2:4].isnan().all() and torch.equal(V.gated_linear(x, w, w)[keep], gate[keep])
        u = w.clone()
        u[5, 11] = math.inf
        y = V.fused_linear(x[keep], u)
        assert torch.equal(y[:, [i for i in range(96) if i != 5]], V.fused_linear(x[keep], w)[:, [i for i in range(96) if i != 5]])
        assert y[:, 5].isnan().all() if len(keep) > 24 else torch.equal(y[:, 5], math.inf * x[keep][:, 11].sign())
