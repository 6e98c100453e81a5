"""How near the dense products come: fp32 operands over fp32's whole range, errors in the 2-norm that the elementwise
bounds of linear_util.py would let pass, and sums that have to come out exactly.

Tolerances, derived before any run.  A dense product of fp32 operands keeps 24 bits of each operand (the pairs of parts that
are left out are below 2^-26 of a product).  64 values at a time are summed in the tensor core, where each of the last four
steps cuts at most 2^-23, 0.35 2^-23 on average, of what it has; the K / 64 sums are then added with rounding (0.2 2^-23 rms of
the running sum, which grows with the root of its length).  For random signs that is sqrt(4^2 0.35^2 + 0.2^2 K / 128) 2^-23 of
the result's 2-norm: 1.7e-7, and 3.4e-7 at K = 20000.  1e-6 is held; operands of two parts instead of three are
2e-6 off at best (2^-18 / sqrt(3) a value, both operands).  The engine of dot products is nearer.

16- and 8-bit operands are summed in the tensor core, which cuts every product to two bits below the running sum's last place:
2^-26 of the running sum at most, half of it on average, and the running sum is sqrt(i / K) of the result: (2/3) K 2^-27.
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
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
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


# ---------------------------------------------------------------------------- errors in the 2-norm
LONG = [1001, 9000, 20000]


@pytest.mark.parametrize("k", LONG)
@pytest.mark.parametrize("m", [1, 8, 24, 30, 300])
def test_fp32_operands_keep_their_bits(m, k):
    """Two parts instead of three are 3.4e-6 off, any one of the six pairs left out at least 2.4e-6 (on CPU, these values)."""
    g = gen(k)
    x, w, u, b = randn(g, m, k), randn(g, 100, k), randn(g, 100, k), randn(g, 100)
    s, t = x.to(F64) @ w.to(F64).t(), x.to(F64) @ u.to(F64).t()
    assert off(V.fused_linear(x, w), s) < 1e-6
    r = randn(g, m, 100)
    assert off(V.fused_linear(x, w, b, activation="relu", residual=r), torch.relu(s + b) + r) < 1e-6
    # (a product of two sums: their errors side by side)
    assert off(V.gated_linear(x, w, u, activation="relu"), torch.relu(s) * t) < 1.5e-6


@pytest.mark.parametrize("m,k,n", [(1001, 60, 300), (200, 60, 9000), (20000, 40, 64), (64, 300, 20000)])
def test_fp32_gradients_keep_their_bits(m, k, n):
    """dx sums over n, dw and the bias over m.  (Gated: dg and du are products of four fp32 values, each sum 2e-7 off.)"""
    g = gen(m)
    x, w, u, b = (t.requires_grad_() for t in (randn(g, m, k), randn(g, n, k) / k ** 0.5, randn(g, n, k) / k ** 0.5, randn(g, n)))
    d = randn(g, m, n)
    x64, w64, u64, d64 = (t.detach().to(F64) for t in (x, w, u, d))
    dx, dw, db = torch.autograd.grad(V.fused_linear(x, w, b), (x, w, b), d)
    assert off(dx, d64 @ w64) < 1e-6 and off(dw, d64.t() @ x64) < 1e-6 and off(db, d64.sum(0)) < 1e-6
    dx, dw, du = torch.autograd.grad(V.gated_linear(x, w, u, activation="relu"), (x, w, u), d)
    a, up = x64 @ w64.t(), x64 @ u64.t()
    pg, pu = torch.where(V.fused_linear(x, w).detach() > 0, d64 * up, 0.0), d64 * torch.relu(a)
    assert off(dx, pg @ w64 + pu @ u64) < 1.5e-6 and off(dw, pg.t() @ x64) < 1.5e-6 and off(du, pu.t() @ x64) < 1.5e-6


@pytest.mark.parametrize("k", LONG)
@pytest.mark.parametrize("m", [3, 30, 150, 300])
@pytest.mark.parametrize("dt", [BF16, F16, torch.float8_e4m3fn])
def test_16_and_8_bit_operands_summed_in_fp32(m, k, dt):
    g = gen(m + k)
    bound = k / 24 * 2.0 ** -23 + 2e-7
    if dt is torch.float8_e4m3fn:
        (x, sx), (w, sw) = fp8_rows(randn(g, m, k)), fp8_rows(randn(g, 100, k))
        got, want = V.fused_linear(x, w, x_scale=sx, w_scale=sw, out_dtype=F32), dequantised(x, sx) @ dequantised(w, sw).t()
    else:
        x, w = randn(g, m, k, dt=dt), randn(g, 100, k, dt=dt)
        got, want = V.fused_linear(x, w, out_dtype=F32), x.to(F64) @ w.to(F64).t()
        a = V.gated_linear(x, w, w, activation="silu", out_dtype=F32)
        # (16 more 2^-24 for the exponential; act'(z) z <= 1.1 act(z) but where act is small)
        assert off(a, act64("silu", want) * want) < 2.5 * bound + 1e-6
    assert off(got, want) < bound


# ---------------------------------------------------------------------------- sums that are exact
def whole(g, most, *shape, dt=F32):
    return torch.randint(-most, most + 1, shape, device="cuda", generator=g).to(F32).to(dt)


def exact_operands(g, dt, m, n, k):
    """Whole numbers, every partial sum of whose products is one below 2^24 (fp32: x of two parts)."""
    if dt is F32:
        return whole(g, 511, m, k), whole(g, 1, n, k)
    if dt is torch.float8_e4m3fn:
        return whole(g, 8, m, k, dt=dt), whole(g, 8, n, k, dt=dt)
    return whole(g, 16, m, k, dt=dt), whole(g, 16, n, k, dt=dt)


@pytest.mark.parametrize("dt", [F32, BF16, F16, torch.float8_e4m3fn])
@pytest.mark.parametrize("m", [1, 3, 20, 40, 150, 300])
@pytest.mark.parametrize("k", [64, 257, 9008, 20000])
def test_whole_numbers_come_out_exactly(dt, m, k):
    """One stage, split or part of the sum lost or counted twice shows."""
    for n in (70, 300):
        g = gen(m + n + k)
        x, w = exact_operands(g, dt, m, n, k)
        ones = torch.ones(max(m, n), device="cuda")
        scales = {"x_scale": ones[:m], "w_scale": ones[:n]} if dt is torch.float8_e4m3fn else {}
        want = x.to(F64) @ w.to(F64).t()
        assert torch.equal(V.fused_linear(x, w, out_dtype=F32, **scales).to(F64), want)
        first = x.to(F32)
        first[:, 0] = 1
        u = torch.zeros(n, k, device="cuda")
        u[:, 0] = 1                                  # the up projection gives 1
        x, u = first.to(dt), u.to(dt)
        want = torch.relu(x.to(F64) @ w.to(F64).t())
        scales = {"x_scale": ones[:m], "gate_scale": ones[:n], "up_scale": ones[:n]} if scales else {}
        assert torch.equal(V.gated_linear(x, w, u, activation="relu", out_dtype=F32, **scales).to(F64), want)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(3, 70, 257), (150, 70, 9008), (300, 130, 1000), (20000, 70, 64), (9000, 33, 131)])
def test_whole_gradients_come_out_exactly(dt, m, k, n):
    g = gen(m + k + n)
    x, w = exact_operands(g, dt, m, n, k)
    b, d = torch.zeros(n, device="cuda", dtype=dt), whole(g, 1, m, n, dt=dt)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(V.fused_linear(*leaves), leaves, d)
    d64, x64, w64 = (t.detach().to(F64) for t in (d, x, w))
    assert torch.equal(dx, (d64 @ w64).to(dt)) and torch.equal(dw, (d64.t() @ x64).to(dt)) and torch.equal(db, d64.sum(0).to(dt))
    u = torch.zeros(n, k, device="cuda", dtype=dt)
    u[:, 0] = 1
    with torch.no_grad():
        x[:, 0] = 1
    dw, = torch.autograd.grad(V.gated_linear(x, w, u, activation="relu"), w, d)
    live = (x.detach().to(F64) @ w64.t() > 0).to(F64)
    assert torch.equal(dw, ((d64 * live).t() @ x.detach().to(F64)).to(dt))


# ---------------------------------------------------------------------------- long sums of one sign
def positive(g, *shape, dt, scale=1.0):
    return ((torch.rand(*shape, device="cuda", generator=g) * 0.5 + 0.5) * scale).to(dt)


def product_in_64(a, b):
    """a bᵀ over a long axis, a piece at a time."""
    return sum(a[:, i:i + (1 << 18)].to(F64) @ b[:, i:i + (1 << 18)].to(F64).t() for i in range(0, a.shape[1], 1 << 18))


@pytest.mark.parametrize("dt", [BF16, F16, torch.float8_e4m3fn])
@pytest.mark.parametrize("m", [3, 64, 170])
def test_long_sums_of_one_sign(dt, m):
    """2^22 positive terms.  The tensor core cuts every product to two bits below the running sum's last place, 2^-26 of it and
    1.4 times that a term on average at most, the running sum being half of the run's: 2^-27 1.4 a term, 3.4e-4 for
    runs of 2^15 and 1.4e-3 for runs of 2^17.  (Unsplit, 2 to 3 in a hundred are gone.)"""
    g = gen(m)
    k, n = 1 << 22, 64
    x, w = positive(g, m, k, dt=dt), positive(g, n, k, dt=dt)
    ones = torch.ones(max(m, n), device="cuda")
    want = product_in_64(x, w)
    scales = {"x_scale": ones[:m], "w_scale": ones[:n]} if dt is torch.float8_e4m3fn else {}
    y = V.fused_linear(x, w, out_dtype=F32, **scales)
    lost = 3.4e-4 if dt is F16 else 1.4e-3
    assert bool(((y.to(F64) - want).abs() <= lost * want).all()), off(y, want)
    scales = {"x_scale": ones[:m], "gate_scale": ones[:n], "up_scale": ones[:n]} if scales else {}
    y = V.gated_linear(x, w, w, activation="relu", out_dtype=F32, **scales)
    assert bool(((y.to(F64) - want * want).abs() <= 2.01 * lost * want * want).all()), off(y, want * want)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_long_gradients_of_one_sign(dt):
    g = gen(5)
    tokens, k, n = 1 << 22, 64, 72
    half, lost = torch.finfo(dt).eps / 2, 3.4e-4 if dt is F16 else 1.4e-3
    x, w = positive(g, tokens, k, dt=dt), positive(g, n, k, dt=dt).requires_grad_()
    d = positive(g, tokens, n, dt=dt, scale=2.0 ** -8)
    want = product_in_64(d.t(), x.t())
    dw, = torch.autograd.grad(V.fused_linear(x, w), w, d)
    assert bool(((dw.to(F64) - want).abs() <= (lost + half) * want).all()), off(dw, want)
    # dx: a wide layer's; the sum runs over n, of a gated block over both weights
    del x, w, d
    x, w = positive(g, 40, k, dt=dt).requires_grad_(), positive(g, 1 << 21, k, dt=dt, scale=2.0 ** -10)
    d = positive(g, 40, 1 << 21, dt=dt, scale=2.0 ** -8)
    dx, = torch.autograd.grad(V.fused_linear(x, w), x, d)
    want = product_in_64(d, w.t())
    assert bool(((dx.to(F64) - want).abs() <= (lost + half) * want).all()), off(dx, want)


# ---------------------------------------------------------------------------- scales whose product leaves fp32's range
@pytest.mark.parametrize("m,k,n", [(1, 4096, 64), (3, 4096, 64), (40, 4096, 2000), (40, 4096, 20000), (300, 4096, 200), (300, 9008, 70)])
@pytest.mark.parametrize("rows,cols", [(1e-25, 1e-20), (1e-20, 1e-25), (1e30, 1e20), (1e20, 1e30), (1e-30, 1e30), (1e30, 1e-30),
                                       (2.0 ** -109, 1e4)])
def test_scales_far_from_1(m, k, n, rows, cols):
    """Sums of up to 8e8, and of 0 in every other row: the result is fp32's where it has one, to the sum's and two
    multiplications' rounding."""
    g = gen(m + n)
    x, w = (torch.randint(1, 9, s, device="cuda", generator=g).float() * 56 for s in ((m, k), (n, k)))
    x[1::2] = 0
    x, w = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    sx, sw = torch.full((m,), rows, device="cuda"), torch.full((n,), cols, device="cuda")
    want = dequantised(x, sx) @ dequantised(w, sw).t()
    y = V.fused_linear(x, w, x_scale=sx, w_scale=sw, out_dtype=F32)
    one = torch.ones_like(sw) / sx[0]
    h = V.gated_linear(x, w, w, activation="relu", x_scale=sx, gate_scale=sw, up_scale=one, out_dtype=F32)
    sums = x.to(F64) @ w.to(F64).t()
    for got, exact in ((y, want), (h, want * sums)):
        over = exact > MOST
        assert bool((got[over] == math.inf).all()) and bool((got[~over].to(F64) - exact[~over]).abs().le(
            4e-6 * exact[~over].abs() + 2.0 ** -126).all())


@pytest.mark.parametrize("dt", [F16, BF16])
def test_long_sums_of_few_rows_and_many_outputs(dt):
    """More tiles of weights than SMs, whose clusters split K because it is long; just below, at and beyond what eight take."""
    g = gen(21)
    for k in ((1 << 15) + 64, 1 << 18, (1 << 18) + 64):
        n, m = (20000 if k < 1 << 17 else 1200), 20
        x, w = whole(g, 4, m, k, dt=dt), whole(g, 4, n, k, dt=dt)
        want = product_in_64(x, w)
        assert torch.equal(V.fused_linear(x, w, out_dtype=F32).to(F64), want)
        u = torch.zeros(n, k, device="cuda", dtype=dt)
        u[:, 0] = 1
        x[:, 0] = 1
        want = torch.relu(product_in_64(x, w))
        assert torch.equal(V.gated_linear(x, w, u, activation="relu", out_dtype=F32).to(F64), want)
        x, w = positive(g, m, k, dt=dt), positive(g, n, k, dt=dt)
        want, lost = product_in_64(x, w), 3.4e-4 if dt is F16 else 1.4e-3
        assert bool(((V.fused_linear(x, w, out_dtype=F32).to(F64) - want).abs() <= lost * want).all())
        del x, w, u, want
