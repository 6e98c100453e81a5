"""The dense products with epilogues (fused_linear, gated_linear), forward and backward, against
formulas in 64 bits (linear_util.py, where the tolerances are derived)."""
import math
import zlib

import pytest
import torch

import verace_v1_b200 as V
from linear_util import (F64, act64, assert_within, dequantised, fp8_rows, gated64, gated_backward64, linear64,
                         linear_backward64, up64)

pytestmark = pytest.mark.gpu
F32, BF16, F16, FP8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
TYPES = [F32, BF16, F16]


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def randn(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def weight(g, n, k, dt=F32, gain=1.0):
    return (gain * torch.randn(n, k, device="cuda", generator=g) / math.sqrt(max(k, 1))).to(dt)


# m around the few-token limits (160; 112 of small gated weights) and the tiles' borders; k and n that no tile or vector divides
SIZES = [(1, 64, 128), (1, 1024, 2048), (2, 72, 129), (7, 1000, 255), (8, 1, 1), (16, 65, 257), (17, 513, 64),
         (33, 100, 1001), (64, 4096, 512), (65, 256, 300), (127, 640, 128), (128, 128, 130), (129, 200, 520),
         (255, 71, 256), (257, 1024, 777), (300, 320, 1024), (1000, 129, 640), (97, 130, 100), (113, 1030, 200),
         (145, 1000, 640), (150, 4100, 1100), (160, 8192, 1000), (161, 8192, 1000)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt", TYPES)
def test_linear(m, k, n, dt):
    g = gen(m, k, n)
    x, w = randn(g, m, k, dt=dt), weight(g, n, k, dt)
    assert_within(V.fused_linear(x, w), linear64(x, w, None, None, None, dt), "plain")
    b, r = randn(g, n, dt=dt), randn(g, m, n, dt=dt)
    assert_within(V.fused_linear(x, w, b, activation="gelu", residual=r), linear64(x, w, b, "gelu", r, dt), "epilogue")


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m", [5, 300])
def test_linear_activations(act, dt, m):
    g = gen(act, m)
    x, w, b = randn(g, m, 96, dt=dt), weight(g, 160, 96, dt, 4.0), randn(g, 160, dt=dt)
    assert_within(V.fused_linear(x, w, b, activation=act), linear64(x, w, b, act, None, dt))
    y = V.fused_linear(x, w, b, activation=act, out_dtype=F32)
    assert y.dtype is F32
    assert_within(y, linear64(x, w, b, act, None, F32))


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt", TYPES)
def test_gated(m, k, n, dt):
    g = gen(m, k, n, 1)
    x, wg, wu = randn(g, m, k, dt=dt), weight(g, n, k, dt, 2.0), weight(g, n, k, dt, 2.0)
    assert_within(V.gated_linear(x, wg, wu), gated64(x, wg, wu, "situ", dt))


@pytest.mark.parametrize("act", ["situ", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m", [5, 300])
def test_gated_activations(act, dt, m):
    g = gen(act, m, 2)
    x, wg, wu = randn(g, m, 96, dt=dt), weight(g, 160, 96, dt, 6.0), weight(g, 160, 96, dt, 6.0)
    assert_within(V.gated_linear(x, wg, wu, activation=act), gated64(x, wg, wu, act, dt))
    y = V.gated_linear(x, wg, wu, activation=act, out_dtype=F32)
    assert y.dtype is F32
    assert_within(y, gated64(x, wg, wu, act, F32))


@pytest.mark.parametrize("m,k,n", SIZES)
def test_8_bits(m, k, n):
    g = gen(m, k, n, 3)
    (x, sx), (wg, sg), (wu, su) = (fp8_rows(t) for t in (randn(g, m, k), weight(g, n, k), weight(g, n, k)))
    x64, g64, u64 = dequantised(x, sx), dequantised(wg, sg), dequantised(wu, su)
    r = randn(g, m, n, dt=BF16)
    y = V.fused_linear(x, wg, x_scale=sx, w_scale=sg, residual=r)
    assert y.dtype is BF16
    assert_within(y, linear64(x64, g64, None, None, r, BF16), "linear")
    for odt in (BF16, F32, F16):
        b = randn(g, n, dt=odt)
        assert_within(V.fused_linear(x, wg, b, activation="silu", x_scale=sx, w_scale=sg, out_dtype=odt),
                      linear64(x64, g64, b, "silu", None, odt), f"linear {odt}")
        h = V.gated_linear(x, wg, wu, x_scale=sx, gate_scale=sg, up_scale=su, out_dtype=odt)
        assert h.dtype is odt
        assert_within(h, gated64(x64, g64, u64, "situ", odt), f"gated {odt}")


@pytest.mark.parametrize("m,k,f", [s for s in SIZES if s[0] * s[2] < 400000])
@pytest.mark.parametrize("dt", TYPES)
def test_gated_backward(m, k, f, dt):
    g = gen(m, k, f, 4)
    x, wg, wu = (t.requires_grad_() for t in (randn(g, m, k, dt=dt), weight(g, f, k, dt, 2.0), weight(g, f, k, dt, 2.0)))
    d = randn(g, m, f, dt=dt)
    h = V.gated_linear(x, wg, wu)
    got = torch.autograd.grad(h, (x, wg, wu), d)
    assert_within(h.detach(), gated64(x.detach(), wg.detach(), wu.detach(), "situ", dt), "out")
    want = gated_backward64(x.detach(), wg.detach(), wu.detach(), "situ", d, dt)
    for name, a, b in zip(("dx", "dw_gate", "dw_up"), got, want):
        assert a.dtype is dt
        assert_within(a, b, name)


@pytest.mark.parametrize("act", ["situ", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt,odt", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
def test_gated_backward_activations(act, dt, odt):
    g = gen(act, 5)
    x, wg, wu = (t.requires_grad_() for t in (randn(g, 150, 80, dt=dt), weight(g, 96, 80, dt, 3.0), weight(g, 96, 80, dt, 3.0)))
    d = randn(g, 150, 96, dt=odt)
    got = torch.autograd.grad(V.gated_linear(x, wg, wu, activation=act, out_dtype=odt), (x, wg, wu), d)
    want = gated_backward64(x.detach(), wg.detach(), wu.detach(), act, d, odt)
    for name, a, b in zip(("dx", "dw_gate", "dw_up"), got, want):
        assert_within(a, b, name)


@pytest.mark.parametrize("m,k,n", [s for s in SIZES if s[0] * s[2] < 400000])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", [None, "silu"])
def test_linear_backward(m, k, n, dt, act):
    g = gen(m, k, n, 6)
    x, w, b, r = (t.requires_grad_() for t in (randn(g, m, k, dt=dt), weight(g, n, k, dt), randn(g, n, dt=dt),
                                               randn(g, m, n, dt=dt)))
    d = randn(g, m, n, dt=dt)
    got = torch.autograd.grad(V.fused_linear(x, w, b, activation=act, residual=r), (x, w, b, r), d)
    want = linear_backward64(x.detach(), w.detach(), b.detach(), act, d, dt)
    for name, a, c in zip(("dx", "dw", "dbias"), got, want):
        assert_within(a, c, name)
    assert torch.equal(got[3], d)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt,odt", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
def test_linear_backward_activations(act, dt, odt):
    g = gen(act, 7)
    x, w, b = (t.requires_grad_() for t in (randn(g, 140, 88, dt=dt), weight(g, 96, 88, dt, 3.0), randn(g, 96, dt=dt)))
    d = randn(g, 140, 96, dt=odt)
    got = torch.autograd.grad(V.fused_linear(x, w, b, activation=act, out_dtype=odt), (x, w, b), d)
    for name, a, c in zip(("dx", "dw", "dbias"), got, linear_backward64(x.detach(), w.detach(), b.detach(), act, d, odt)):
        assert_within(a, c, name)


def test_gradients_against_differences():
    """fp32 gradients against central differences of the fp32 forward along random directions.  A step s leaves
    s^2 / 6 times the third derivative of sum d a(g) b(u), at most 8 (1 + |a| + |b|) (|g'| + |u'|)^3 a term (the
    factor over the values' third derivatives, all below 2, holds along the whole step), and the forward's rounding."""
    g = gen(8)
    x, wg, wu = randn(g, 6, 40), weight(g, 50, 40), weight(g, 50, 40)
    d = randn(g, 6, 50)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(V.gated_linear(*leaves), leaves, d)
    s = 2.0 ** -6
    a, b = act64("situ", x.double() @ wg.double().t()).abs(), up64("situ", x.double() @ wu.double().t()).abs()
    _, rounding = gated64(x, wg, wu, "situ", F32)
    for i in range(3):
        for _ in range(5):
            v = torch.randn(leaves[i].shape, device="cuda", generator=g)
            v = v / v.norm()
            ends = []
            for sign in (1, -1):
                t = [x, wg, wu]
                t[i] = t[i] + sign * s * v
                ends.append((V.gated_linear(*t).double() * d.double()).sum())
            moved = ((v @ wg.t()).abs() + (v @ wu.t()).abs() if i == 0 else (x @ v.t()).abs()).double()
            tol = (d.double().abs() * (s * s / 6 * 8 * (1 + a + b) * moved ** 3 + 2 * rounding / s)).sum()
            got = (grads[i].double() * v.double()).sum()
            assert abs(float((ends[0] - ends[1]) / (2 * s) - got)) < float(tol)


def test_only_the_gradients_asked_for():
    g = gen(9)
    x, wg, wu = randn(g, 20, 64, dt=BF16), weight(g, 96, 64, BF16), weight(g, 96, 64, BF16)
    d = randn(g, 20, 96, dt=BF16)
    full = [t.clone().requires_grad_() for t in (x, wg, wu)]
    want = torch.autograd.grad(V.gated_linear(*full), full, d)
    for i in range(3):
        t = [x, wg, wu]
        t[i] = t[i].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(V.gated_linear(*t), t[i], d)[0], want[i])
    w, b, r = weight(g, 96, 64, BF16).requires_grad_(), randn(g, 96, dt=BF16).requires_grad_(), randn(g, 20, 96, dt=BF16)
    y = V.fused_linear(x, w.detach(), b, residual=r)
    assert_within(torch.autograd.grad(y, b, d)[0], linear_backward64(x, w.detach(), b.detach(), None, d, BF16)[2])
    r = r.requires_grad_()
    y = V.fused_linear(x, w.detach(), residual=r)
    assert torch.equal(torch.autograd.grad(y, r, d)[0], d)


def test_expanded_gradient_and_repeated_inputs():
    """The gradient of a sum is an expanded tensor; one weight as gate and up gets both gradients."""
    g = gen(10)
    x, w = randn(g, 9, 33).requires_grad_(), weight(g, 40, 33).requires_grad_()
    got = torch.autograd.grad(V.gated_linear(x, w, w, activation="silu").sum(), (x, w))
    want = gated_backward64(x.detach(), w.detach(), w.detach(), "silu", torch.ones(9, 40, device="cuda"), F32)
    assert_within(got[0], want[0])
    assert_within(got[1], (want[1][0] + want[2][0], want[1][1] + want[2][1] + 2.0 ** -24 * (want[1][0] + want[2][0]).abs()))


@pytest.mark.parametrize("m,k,n", [(0, 64, 32), (3, 64, 0), (3, 0, 32), (0, 0, 0)])
@pytest.mark.parametrize("dt", TYPES)
def test_empty(m, k, n, dt):
    g = gen(11)
    x, w, b = randn(g, m, k, dt=dt), torch.zeros(n, k, device="cuda", dtype=dt), randn(g, n, dt=dt)
    y = V.fused_linear(x, w, b, activation="silu")
    assert y.shape == (m, n)
    assert_within(y, linear64(x, w, b, "silu", None, dt))
    assert_within(V.gated_linear(x, w, w), gated64(x, w, w, "situ", dt))
    x, w = x.requires_grad_(), w.requires_grad_()
    for out in (V.fused_linear(x, w, b), V.gated_linear(x, w, w)):
        dx, dw = torch.autograd.grad(out, (x, w), torch.ones_like(out))
        assert dx.shape == x.shape and dw.shape == w.shape and not dx.any() and not dw.any()


def test_leading_dimensions():
    g = gen(12)
    x, w, r = randn(g, 2, 3, 5, 64, dt=BF16), weight(g, 48, 64, BF16), randn(g, 2, 3, 5, 48, dt=BF16)
    y = V.fused_linear(x, w, residual=r)
    assert y.shape == (2, 3, 5, 48)
    assert torch.equal(y.view(30, 48), V.fused_linear(x.view(30, 64), w, residual=r.view(30, 48)))
    one = V.gated_linear(x[0, 0, 0], w, w)
    assert one.shape == (48,)
    assert_within(one[None], gated64(x[0, 0, 0][None], w, w, "situ", BF16))


@pytest.mark.parametrize("dt", TYPES + [FP8])
@pytest.mark.parametrize("m", [3, 200])
def test_strides_and_alignment(dt, m):
    """Rows inside wider tensors, off 16-byte borders, transposed and repeated: the result is that of dense operands."""
    g = gen(13)
    k, n = 136, 72
    odt = BF16 if dt is FP8 else dt
    big_x = randn(g, m + 2, k + 40).to(dt)
    big_w = weight(g, n + 2, k + 40).to(dt)
    sx, sw = torch.rand(m, device="cuda", generator=g) + 0.5, torch.rand(n, device="cuda", generator=g) + 0.5
    scales = {"x_scale": sx, "w_scale": sw} if dt is FP8 else {}
    gscales = {"x_scale": sx, "gate_scale": sw, "up_scale": sw} if dt is FP8 else {}

    def byte(t):    # (float8 tensors are moved about as bytes)
        return t.view(torch.uint8) if dt is FP8 else t

    def dense(t):
        return byte(t).contiguous().view(dt) if dt is FP8 else t.contiguous()

    forms = [(big_x[1:m + 1, 16:16 + k], big_w[:n, 32:32 + k]), (big_x[1:m + 1, 3:3 + k], big_w[1:n + 1, 5:5 + k]),
             (byte(dense(big_x[:m, :k])).t().contiguous().t().view(dt) if dt is FP8 else big_x[:m, :k].t().contiguous().t(),
              big_w[:n, :k]),
             (byte(big_x)[:1, :k].expand(m, k).view(dt), big_w[:n, 1:1 + k])]
    r = randn(g, m, 2 * n, dt=odt)
    for x, w in forms:
        want = V.fused_linear(dense(x), dense(w), residual=r[:, n:].contiguous(), **scales)
        assert torch.equal(V.fused_linear(x, w, residual=r[:, n:], **scales), want)
        assert torch.equal(V.fused_linear(x, w, residual=r[:, n:].t().contiguous().t(), **scales), want)
        want = V.gated_linear(dense(x), dense(w), dense(w), **gscales)
        assert torch.equal(V.gated_linear(x, w, dense(w), **gscales), want)
    if dt is not FP8:
        for x, w in forms[:3]:
            a = [dense(x).requires_grad_(), dense(w).requires_grad_()]
            b = [x.detach().requires_grad_(), w.detach().requires_grad_()]
            d = randn(g, m, n, dt=dt)
            ga = torch.autograd.grad(V.fused_linear(*a, activation="silu"), a, d)
            gb = torch.autograd.grad(V.fused_linear(*b, activation="silu"), b, d.t().contiguous().t())
            assert all(torch.equal(u, v) for u, v in zip(ga, gb))
            ga = torch.autograd.grad(V.gated_linear(a[0], a[1], a[1]), a, d)
            gb = torch.autograd.grad(V.gated_linear(b[0], b[1], b[1]), b, d)
            assert all(torch.equal(u, v) for u, v in zip(ga, gb))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m", [4, 260])
def test_special_values(dt, m):
    """A NaN in one row of x reaches that row only; large sums saturate as the formulas do."""
    g = gen(14)
    x, w = randn(g, m, 64, dt=dt), weight(g, 96, 64, dt)
    want, gate = V.fused_linear(x, w), V.gated_linear(x, w, w)
    bad = x.clone()
    bad[1, 5] = math.nan
    bad[2, 7] = math.inf
    y, h = V.fused_linear(bad, w), V.gated_linear(bad, w, w)
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[keep], want[keep]) and torch.equal(h[keep], gate[keep])
    assert y[1].isnan().all() and h[1].isnan().all() and not y[2].isfinite().any()
    big = (x.float() * 200).to(dt)
    for act in ("situ", "silu", "gelu", "gelu_tanh", "relu"):
        assert_within(V.gated_linear(big, w, w, activation=act, out_dtype=F32), gated64(big, w, w, act, F32), act)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_repeatable_and_out_is_not_shared(m):
    """The same bits on every call, also when calls overlap on two streams."""
    g = gen(15)
    x, wg, wu = randn(g, m, 512, dt=BF16), weight(g, 700, 512, BF16), weight(g, 700, 512, BF16)
    d = randn(g, m, 700, dt=BF16)

    def call():
        t = [v.detach().requires_grad_() for v in (x, wg, wu)]
        h = V.gated_linear(*t)
        return (h.detach(),) + torch.autograd.grad(h, t, d)
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            out.append(call())
    torch.cuda.synchronize()
    for o in out:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_engines_side_by_side_on_streams():
    """Products of every engine and of the largest claims on an SM's memory, on four streams at once: their bits alone."""
    g = gen(26)
    x, wg, wu = randn(g, 160, 1024, dt=BF16), weight(g, 4224, 1024, BF16), weight(g, 4224, 1024, BF16)
    (x8, sx), (w8, sg), (u8, su) = (fp8_rows(t) for t in (randn(g, 150, 4096), weight(g, 1100, 4096), weight(g, 1100, 4096)))
    small, w7, r7 = randn(g, 7, 2048, dt=F16), weight(g, 512, 2048, F16), randn(g, 7, 512, dt=F16)
    big, wb = randn(g, 600, 512, dt=BF16), weight(g, 1000, 512, BF16)
    one, w1 = randn(g, 1, 256, dt=F32), weight(g, 512, 256, F32)
    calls = [lambda: V.gated_linear(x, wg, wu), lambda: V.fused_linear(small, w7, residual=r7), lambda: V.fused_linear(big, wb),
             lambda: V.fused_linear(one, w1), lambda: V.fused_linear(x, wg, activation="silu"),
             lambda: V.gated_linear(x8, w8, u8, x_scale=sx, gate_scale=sg, up_scale=su)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, out = [torch.cuda.Stream() for _ in range(4)], []
    for i in range(10):
        for s, st in enumerate(streams):
            for j in range(len(calls)):
                which = (i + s + j) % len(calls)
                with torch.cuda.stream(st):
                    out.append((which, calls[which]()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in out)


@pytest.mark.parametrize("m", [2, 120, 200])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_captured_in_a_graph(m, dt):
    """Forward and backward captured once and replayed on new values; two graphs do not disturb each other."""
    g = gen(16)
    k, f = 256, 300
    x, wg, wu, w = randn(g, m, k, dt=dt), weight(g, f, k, dt), weight(g, f, k, dt), weight(g, k, f, dt)
    d = randn(g, m, k, dt=dt)

    def block(x):
        t = [v.detach().requires_grad_() for v in (x, wg, wu, w)]
        y = V.fused_linear(V.gated_linear(t[0], t[1], t[2]), t[3], residual=t[0])
        return (y.detach(),) + torch.autograd.grad(y, t, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, ins = [], [], []
    for i in range(2):
        ins.append(x.clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(block(ins[-1]))
        graphs.append(graph)
    for i, t in enumerate(ins):
        t.copy_(randn(g, m, k, dt=dt))
    for i in (0, 1, 0):
        graphs[i].replay()
    torch.cuda.synchronize()
    for t, o in zip(ins, outs):
        for a, b in zip(o, block(t)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_between_streams_and_copies(m):
    """In a graph behind a copy, a join of two streams and kernels of torch's own."""
    g = gen(m, 24)
    x, w, w2 = randn(g, m, 128, dt=BF16), weight(g, 128, 128, BF16), weight(g, 128, 128, BF16)
    norm = torch.nn.RMSNorm(128, eps=1e-6, device="cuda", dtype=BF16).requires_grad_(False)
    into, side = torch.empty_like(x), torch.cuda.Stream()

    def work():
        into.copy_(x)
        a = V.fused_linear(into, w)
        here, there = torch.cuda.Event(), torch.cuda.Event()
        here.record()
        with torch.cuda.stream(side):
            side.wait_event(here)
            b = V.gated_linear(a, w, w2)
            there.record()
        c = V.fused_linear(a, w2, activation="silu")
        torch.cuda.current_stream().wait_event(there)
        q, s = V.add_rmsnorm_fp8(c, b, norm)
        y = V.fused_linear(c + b, w, residual=b)
        return a, b, c, y, q.view(torch.uint8), s
    first = torch.cuda.Stream()
    first.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(first):
        work()
    torch.cuda.current_stream().wait_stream(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    x.copy_(randn(g, m, 128, dt=BF16))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    kept = [t.clone() for t in got]
    want = work()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_rows_behind_the_output_stay():
    """Nothing is written outside of the output: its allocation's neighbours keep their values."""
    g = gen(17)
    for m, k, n in [(3, 64, 33), (130, 72, 131), (257, 64, 259)]:
        x, wg, wu = randn(g, m, k, dt=BF16), weight(g, n, k, BF16), weight(g, n, k, BF16)
        L = V._lib.lib()
        flat = torch.full((m * n + 512,), 7.0, device="cuda", dtype=BF16)
        nws = L.verace_gated_linear_workspace(m, n, k, 1)
        ws = torch.empty(max(nws, 1), dtype=torch.uint8, device="cuda")
        out = flat[256:256 + m * n]
        rc = L.verace_gated_linear(x.data_ptr(), k, None, wg.data_ptr(), wu.data_ptr(), k, None, None, out.data_ptr(), None,
                                   None, m, n, k, 5, 4.0, 25.0, 1, 1, ws.data_ptr(), nws,
                                   torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(out.view(m, n), V.gated_linear(x, wg, wu))
        assert (flat[:256] == 7).all() and (flat[256 + m * n:] == 7).all()


@pytest.mark.parametrize("m", [1, 50, 400])
def test_feed_forward_sub_layer(m):
    """The operators together, as a block uses them: norm with residual to 8 bits, gated product, down projection
    with the residual in its epilogue.  Each step is checked on the step before's own output."""
    g = gen(18)
    k, f = 320, 640
    norm = torch.nn.RMSNorm(k, eps=1e-6, device="cuda", dtype=BF16).requires_grad_(False)
    h, y = randn(g, m, k, dt=BF16), randn(g, m, k, dt=BF16)
    (wg, sg), (wu, su), (wd, sd) = (fp8_rows(t) for t in (weight(g, f, k), weight(g, f, k), weight(g, k, f)))
    h0 = h.clone()
    q, s, n = V.add_rmsnorm_fp8(h, y, norm, return_norm=True)
    assert torch.equal(h, h0 + y)
    a = V.gated_linear(q, wg, wu, x_scale=s, gate_scale=sg, up_scale=su)
    assert_within(a, gated64(dequantised(q, s), dequantised(wg, sg), dequantised(wu, su), "situ", BF16))
    qa, sa = V.quantize_fp8(a)
    out = V.fused_linear(qa, wd, residual=h, x_scale=sa, w_scale=sd)
    assert_within(out, linear64(dequantised(qa, sa), dequantised(wd, sd), None, None, h, BF16))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(300, 9000, 100), (260, 4100, 33), (97, 20000, 64)])
def test_long_sums_over_few_tiles(m, k, n, dt):
    """K is split over many tiles' worth of CTAs, forward and (K the tokens) in the weights' gradients."""
    g = gen(m, k, n, 20)
    x, wg, wu = randn(g, m, k, dt=dt), weight(g, n, k, dt), weight(g, n, k, dt)
    b, r = randn(g, n, dt=dt), randn(g, m, n, dt=dt)
    assert_within(V.fused_linear(x, wg, b, activation="silu", residual=r), linear64(x, wg, b, "silu", r, dt), "linear")
    assert_within(V.gated_linear(x, wg, wu), gated64(x, wg, wu, "situ", dt), "gated")
    # tokens and widths change places
    xt, w1, w2, d = randn(g, k, 40, dt=dt), weight(g, n, 40, dt), weight(g, n, 40, dt), randn(g, k, n, dt=dt)
    leaves = [v.requires_grad_() for v in (xt, w1, w2)]
    got = torch.autograd.grad(V.gated_linear(*leaves, activation="silu"), leaves, d)
    for name, a, c in zip(("dx", "dw_gate", "dw_up"), got, gated_backward64(*(v.detach() for v in leaves), "silu", d, dt)):
        assert_within(a, c, name)
    only = w2.detach().requires_grad_()         # one of the weights alone
    one = torch.autograd.grad(V.gated_linear(xt.detach(), w1.detach(), only, activation="silu"), only, d)[0]
    assert_within(one, gated_backward64(xt.detach(), w1.detach(), only.detach(), "silu", d, dt)[2], "dw_up alone")
    got = torch.autograd.grad(V.fused_linear(xt, w1), (xt, w1), d)
    for name, a, c in zip(("dx", "dw"), got, linear_backward64(xt.detach(), w1.detach(), None, None, d, dt)):
        assert_within(a, c, name)


def test_long_sums_in_8_bits():
    g = gen(21)
    (x, sx), (wg, sg), (wu, su) = (fp8_rows(t) for t in (randn(g, 300, 9008), weight(g, 100, 9008), weight(g, 100, 9008)))
    x64, g64, u64 = dequantised(x, sx), dequantised(wg, sg), dequantised(wu, su)
    b = randn(g, 100, dt=F16)
    assert_within(V.fused_linear(x, wg, b, activation="gelu", x_scale=sx, w_scale=sg, out_dtype=F16),
                  linear64(x64, g64, b, "gelu", None, F16))
    assert_within(V.gated_linear(x, wg, wu, x_scale=sx, gate_scale=sg, up_scale=su), gated64(x64, g64, u64, "situ", BF16))


@pytest.mark.parametrize("m", [1, 3, 50, 300])
@pytest.mark.parametrize("n", [64, 101])
def test_out_may_be_the_residual(m, n):
    """The C entry point with the output in the residual's place, in each engine."""
    g = gen(m, n, 22)
    for dt, code in ((F32, 0), (BF16, 1)):
        x, w, r = randn(g, m, 96, dt=dt), weight(g, n, 96, dt), randn(g, m, n, dt=dt)
        want = V.fused_linear(x, w, residual=r)
        L = V._lib.lib()
        nws = L.verace_linear_workspace(m, n, 96, code)
        ws = torch.empty(max(nws, 1), dtype=torch.uint8, device="cuda")
        rc = L.verace_linear(x.data_ptr(), 96, None, w.data_ptr(), 96, None, None, r.data_ptr(), n, r.data_ptr(), None, m, n, 96,
                             0, code, code, ws.data_ptr(), nws, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(r, want)


@pytest.mark.parametrize("m", [1, 2, 40, 130, 300])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_chains_of_calls_wait_for_each_other(m, dt):
    """Kernels that become resident before the one ahead of them ends: a chain without a wait on the host gives the bits
    of the same chain with one after every call.  The framework's other early launches (rmsnorm, int4) are among them."""
    g = gen(m, 23)
    k, f = 128, 256
    norm = torch.nn.RMSNorm(k, eps=1e-6, device="cuda", dtype=dt).requires_grad_(False)
    wg, wu, wd, w4 = weight(g, f, k, dt), weight(g, f, k, dt), weight(g, k, f, dt), weight(g, k, k, dt)
    q8, s8 = V.quantize_fp8(weight(g, k, k))
    q4, s4, _ = V.quantize_int4(w4)
    first = randn(g, m, k, dt=dt)

    def chain(wait):
        h, out = first.clone(), []
        for _ in range(12):
            n = V.rmsnorm(h, norm)
            wait()
            a = V.gated_linear(n, wg, wu)
            wait()
            h = V.fused_linear(a, wd, residual=h)
            wait()
            q, s = V.add_rmsnorm_fp8(h, n, norm)
            wait()
            y = V.fused_linear(q, q8, x_scale=s, w_scale=s8, out_dtype=dt)
            wait()
            h = V.add_rmsnorm(h, y, out_norm=norm) + V.int4_linear(y, q4, s4)
            wait()
            out.append(h)
        return out
    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))


def test_refusals():
    g = gen(19)
    x, w = randn(g, 4, 64, dt=BF16), weight(g, 32, 64, BF16)
    q, s = V.quantize_fp8(x)
    wq, ws = V.quantize_fp8(w)
    with pytest.raises(ValueError, match="activation"):
        V.fused_linear(x, w, activation="situ")
    with pytest.raises(ValueError, match="activation"):
        V.gated_linear(x, w, w, activation=None)
    with pytest.raises(ValueError, match="beta"):
        V.gated_linear(x, w, w, beta1=0.0)
    with pytest.raises(AssertionError, match="weights"):
        V.fused_linear(x, w[:, :32])
    with pytest.raises(AssertionError, match="weights"):
        V.gated_linear(x, w, w[:16])
    with pytest.raises(AssertionError, match="weights"):
        V.fused_linear(x, w.float())
    with pytest.raises(AssertionError, match="weights"):
        V.fused_linear(x, w.cpu())
    with pytest.raises(AssertionError, match="two dimensions"):
        V.gated_linear(x, w[0], w[0])
    with pytest.raises(ValueError, match="scales"):
        V.fused_linear(q, wq, x_scale=s)
    with pytest.raises(ValueError, match="scales"):
        V.fused_linear(x, w, x_scale=s, w_scale=ws)
    with pytest.raises(AssertionError, match="x_scale"):
        V.fused_linear(q, wq, x_scale=s[:2], w_scale=ws)
    with pytest.raises(ValueError, match="out_dtype"):
        V.fused_linear(x, w, out_dtype=F16)
    with pytest.raises(AssertionError, match="bias"):
        V.fused_linear(x, w, torch.zeros(1, device="cuda", dtype=BF16))
    with pytest.raises(AssertionError, match="residual"):
        V.fused_linear(x, w, residual=torch.zeros(1, 32, device="cuda", dtype=BF16))
    with pytest.raises(AssertionError, match="residual"):
        V.fused_linear(x, w, residual=torch.zeros(4, 32, device="cuda"))
    with pytest.raises(RuntimeError, match="no_grad"):
        V.fused_linear(q, wq, x_scale=s, w_scale=ws, residual=torch.zeros(4, 32, device="cuda", dtype=BF16, requires_grad=True))
    with pytest.raises(ValueError, match="inputs"):
        V.fused_linear(x.double(), w.double())
    t = [v.clone().requires_grad_() for v in (x, w)]
    first = torch.autograd.grad(V.fused_linear(*t), t, torch.ones(4, 32, device="cuda", dtype=BF16), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first[0].sum(), t[0])
    assert V.device_status() == 0
