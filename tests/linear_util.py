"""Formulas of the dense products in 64 bits, with how far a kernel may be from them (imported only
by tests).

Tolerances, derived before any run.  e = eps / 2 of the type is the relative error of one rounding.
A sum of k products in fp32, in any order and with each addition rounded or cut to 24 bits, is off by
at most (k + 8) 2^-23 sum |x| |w|; the 8 covers scales and bias, and for fp32 operands the three bf16
parts, whose dropped terms are below 2^-23 of each product.  The 16-bit types' activations (approximate exponentials and reciprocals, a
few 2^-22 each) are held to 2^-18 of their value, the fp32 ones to 2^-20.  Slopes: |act'| <= 2,
|act''| <= 1.2 for every activation here (relu but for its border), |up'| <= 1, |up''| <= 0.1.
"""
import math

import torch

F64, F32 = torch.float64, torch.float32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
B1, B2 = 4.0, 25.0


def tiny(dt):
    """Half the step of the type's subnormal numbers."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def act64(name, z):
    if name is None:
        return z
    if name == "relu":
        return torch.relu(z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return B1 * torch.tanh(z / B1) / (1 + torch.exp(-z))


def up64(name, u):
    return B2 * torch.tanh(u / B2) if name == "situ" else u


def product64(x, w):
    """(x wᵀ, the bound of its fp32 sum's error)."""
    x, w = x.to(F64), w.to(F64)
    return x @ w.t(), (x.shape[1] + 8) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def act_error(dt):
    return 2.0 ** -20 if dt is torch.float32 else 2.0 ** -18


def linear64(x, w, bias, act, residual, odt):
    """(out, its tolerance) of fused_linear on these values."""
    z, tol = product64(x, w)
    if bias is not None:
        z = z + bias.to(F64)
        tol = tol + 2.0 ** -22 * bias.to(F64).abs()
    a = act64(act, z)
    tol = 2 * tol + act_error(odt) * (a.abs() + 1e-6 * z.abs())
    y = a
    if residual is not None:
        y = y + residual.to(F64)
        tol = tol + 2.0 ** -23 * (a.abs() + residual.to(F64).abs())
    return y, tol + HALF[odt] * (y.abs() + tol) + tiny(odt)


def gated64(x, wg, wu, act, odt):
    g, tg = product64(x, wg)
    u, tu = product64(x, wu)
    a, b = act64(act, g), up64(act, u)
    tol = 2 * tg * (b.abs() + tu) + a.abs() * tu + 3 * act_error(odt) * (a * b).abs() + 1e-6 * act_error(odt)
    return a * b, tol + HALF[odt] * ((a * b).abs() + tol) + tiny(odt)


def slopes64(f, z):
    z = z.detach().requires_grad_()
    return torch.autograd.grad(f(z).sum(), z)[0]


def gated_backward64(x, wg, wu, act, d, odt):
    """[(gradient, tolerance)] of x, w_gate, w_up: the sums are kept in fp32, dg and du are rounded to x's
    type before they enter the products."""
    dt, e, es = x.dtype, HALF[x.dtype], HALF[F32]
    x, wg, wu, d = (t.to(F64) for t in (x, wg, wu, d))
    g, tg = product64(x, wg)
    u, tu = product64(x, wu)
    tg, tu = tg + es * g.abs(), tu + es * u.abs()
    a, b = act64(act, g), up64(act, u)
    da, db = slopes64(lambda z: act64(act, z), g), slopes64(lambda z: up64(act, z), u)
    dg, du = d * da * b, d * a * db
    soft = 0.0 if act == "relu" else 1.2
    t_dg = d.abs() * (soft * tg * (b.abs() + tu) + 2 * tu) + (e + 4 * act_error(odt)) * d.abs() * 2 * b.abs() + tiny(dt)
    t_du = d.abs() * (2 * tg + (a.abs() + 2 * tg) * 0.1 * tu) + (e + 4 * act_error(odt)) * d.abs() * a.abs() + tiny(dt) \
        + 4 * act_error(odt) * d.abs()
    # (e |dg| with |dg| <= |d| 2 |b|, and the derivative's own cancelling terms, each at most 2 |b|)
    def out(v, t):
        return v, t + e * (v.abs() + t) + tiny(dt)
    m, f = g.shape
    k = x.shape[1]
    sx = (2 * f + 8) * 2.0 ** -23 * ((dg.abs() + t_dg) @ wg.abs() + (du.abs() + t_du) @ wu.abs())
    sw = (m + 8) * 2.0 ** -23
    return [out(dg @ wg + du @ wu, t_dg @ wg.abs() + t_du @ wu.abs() + sx),
            out(dg.t() @ x, t_dg.t() @ x.abs() + sw * ((dg.abs() + t_dg).t() @ x.abs())),
            out(du.t() @ x, t_du.t() @ x.abs() + sw * ((du.abs() + t_du).t() @ x.abs()))]


def linear_backward64(x, w, bias, act, d, odt):
    """[(gradient, tolerance)] of x, w, bias."""
    dt, e, es = x.dtype, HALF[x.dtype], HALF[F32]
    x, w, d = (t.to(F64) for t in (x, w, d))
    z, tz = product64(x, w)
    if bias is not None:
        z = z + bias.to(F64)
    tz = 2 * tz + es * z.abs()
    p = d * slopes64(lambda v: act64(act, v), z)
    soft = 0.0 if act in (None, "relu") else 1.2
    tp = d.abs() * (soft * tz + (0.0 if act in (None, "relu") else 8 * act_error(odt))) + e * p.abs() + tiny(dt)
    m, n = z.shape

    def out(v, t, terms, mass):
        t = t + (terms + 8) * 2.0 ** -23 * mass
        return v, t + e * (v.abs() + t) + tiny(dt)
    q = p.abs() + tp
    return [out(p @ w, tp @ w.abs(), n, q @ w.abs()), out(p.t() @ x, tp.t() @ x.abs(), m, q.t() @ x.abs()),
            out(p.sum(0), tp.sum(0), m, q.sum(0))]


def assert_within(got, want, what=""):
    """got within the tolerance of (value, tolerance), infinities and NaN where they are."""
    value, tol = want
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)} for {tuple(value.shape)}"
    if got.numel() == 0:
        return
    off = (got.to(F64) - value).abs() - tol
    worst = int(torch.argmax(torch.nan_to_num(off, nan=math.inf)))
    assert bool((off <= 0).all()), (f"{what}: value {worst} is {float(got.reshape(-1)[worst])}, expected "
                                    f"{float(value.reshape(-1)[worst])} within {float(tol.reshape(-1)[worst])}; "
                                    f"{int((~(off <= 0)).sum())} of {got.numel()} are off")


def fp8_rows(t):
    """Rows of t as (e4m3, fp32 scales)."""
    s = t.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100) / 448
    return (t / s).to(torch.float8_e4m3fn), s[:, 0].contiguous()


def dequantised(q, s):
    return q.to(F64) * s.to(F64)[:, None]
