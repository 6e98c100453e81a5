"""RMS norm with the residual's addition and an 8-bit output, against formulas in 64 bits.

Tolerances, derived before any run: the sum h + y is one fp32 addition, rounded to the type: exact.
With n in 64 bits, the kernel's fp32 norm is within (cols / 32 + 40) 2^-24 + 2^-22 of it (a thread's
32 squares or cols / 32 of a row, the joins, rsqrt and three products), its scale likewise; an 8-bit value is within half an
e4m3 step of n / scale: 2^-4 of it, or 2^-10 below 2^-6, plus that error.  ``n`` in the type: one rounding more."""
import math

import pytest
import torch

import verace_v1_b200 as V
from linear_util import HALF, tiny

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def data(rows, cols, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1000 * rows + cols + seed)
    h = (torch.randn(rows, cols, device="cuda", generator=g) * (0.2 + 3 * torch.rand(rows, 1, device="cuda", generator=g))).to(dt)
    y = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    norm = torch.nn.RMSNorm(cols, eps=1e-6, device="cuda", dtype=dt).requires_grad_(False)
    norm.weight.copy_(1 + 0.3 * torch.randn(cols, device="cuda", generator=g))
    return h, y, norm


def check(h, norm, q, scale, n=None):
    """q, scale (and n) of the rows h, which the norm (None: the quantiser) reads."""
    x = h.double()
    rel = 0.0
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + norm.eps).sqrt()
        if norm.weight is not None:
            x = x * norm.weight.double()
        rel = (h.shape[-1] / 32 + 40) * 2.0 ** -24 + 2.0 ** -22
    top = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    s = top / 448
    assert q.dtype is torch.float8_e4m3fn and q.shape == h.shape
    assert scale.dtype is torch.float32 and scale.shape == h.shape[:-1]
    assert ((scale.double() - s[..., 0]).abs() <= (rel + 2.0 ** -22) * s[..., 0]).all()
    v = x / s
    off = (q.double() - v).abs()
    assert (off <= torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + (2 * rel + 2.0 ** -21) * v.abs()).all()
    if n is not None:
        e = HALF[h.dtype]
        assert ((n.double() - x).abs() <= (rel + e * (1 + rel)) * x.abs() + tiny(h.dtype)).all()


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 1000), (9, 1024), (4, 1025), (3, 1032), (2, 4096), (3, 4097), (2, 5001),
          (2, 16384), (1, 16385), (2, 20000), (1, 32768), (700, 256), (333, 4096),
          (3, 5120), (2, 5121), (2, 6143), (3, 7168), (2, 8185), (2, 10240), (2, 12281), (1, 20473), (1, 24576)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dt", TYPES)
def test_norm_to_8_bits(rows, cols, dt):
    h, y, norm = data(rows, cols, dt)
    check(h, norm, *V.rmsnorm_fp8(h, norm))
    check(h, norm, *V.rmsnorm_fp8(h, norm, return_norm=True))
    check(h, None, *V.quantize_fp8(h))
    want = (h.float() + y.float()).to(dt)
    into = torch.full_like(h, math.nan)
    before = h.clone()
    q, s, n = V.add_rmsnorm_fp8(h, y, norm, out=into, return_norm=True)
    assert torch.equal(into, want) and torch.equal(h, before)
    check(want, norm, q, s, n)
    q2, s2 = V.add_rmsnorm_fp8(h, y, norm)          # in place
    assert torch.equal(h, want) and torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))


@pytest.mark.parametrize("dt", TYPES)
def test_norm_without_weight_and_leading_dimensions(dt):
    h, _, _ = data(24, 96, dt)
    norm = torch.nn.RMSNorm(96, elementwise_affine=False, device="cuda")
    q, s = V.rmsnorm_fp8(h.view(2, 3, 4, 96), norm)
    assert q.shape == (2, 3, 4, 96) and s.shape == (2, 3, 4)
    norm.eps = torch.finfo(dt).eps
    check(h, norm, q.view(24, 96), s.view(24))


@pytest.mark.parametrize("cols", [64, 100, 2048, 6000])
@pytest.mark.parametrize("dt", TYPES)
def test_rows_of_zeros_small_values_and_special_ones(cols, dt):
    h, _, norm = data(6, cols, dt)
    h[0] = 0
    h[1] = 0
    h[1, cols // 2] = torch.finfo(dt).smallest_normal
    h[3, 3] = math.nan
    h[4, 5] = math.inf
    q, s = V.quantize_fp8(h)
    assert not q[0].float().any() and abs(float(s[0]) * 448 * 2.0 ** 100 - 1) <= 2.0 ** -23   # (one division in fp32)
    ok = [0, 1, 2, 5]
    check(h[ok], None, q.view(torch.uint8)[ok].view(torch.float8_e4m3fn), s[ok])
    assert s[3].isnan() and q[3].float().isnan().all()          # a NaN takes its row
    assert s[4].isinf() and q[4].float()[5].isnan()
    q, s = V.rmsnorm_fp8(h, norm)
    check(h[ok], norm, q.view(torch.uint8)[ok].view(torch.float8_e4m3fn), s[ok])
    assert s[3].isnan() and s[4].isnan()


@pytest.mark.parametrize("dt", TYPES)
def test_misaligned_rows_and_aliases(dt):
    flat = torch.randn(3 * 1024 + 1, device="cuda").to(dt)
    h = flat[1:].view(3, 1024)
    a, b = V.quantize_fp8(h), V.quantize_fp8(h.clone())
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    t = h.t()                       # not contiguous
    a, b = V.quantize_fp8(t), V.quantize_fp8(t.contiguous())
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    _, _, norm = data(3, 1024, dt)
    y = torch.randn(3, 1024, device="cuda").to(dt)
    want = V.add_rmsnorm_fp8(h, y, norm, out=torch.empty_like(y))
    got = V.add_rmsnorm_fp8(h, y, norm, out=y)      # the sum in y's place
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    twice = V.add_rmsnorm_fp8(h, h, norm, out=torch.empty_like(y))
    check((h.float() + h.float()).to(dt), norm, *twice)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", [13, 1017, 1018, 4090, 5001, 32761])
def test_rows_anywhere_in_a_word(dt, cols):
    """Every tensor off the others' alignment; nothing is written beside the outputs."""
    g = torch.Generator(device="cuda").manual_seed(cols)

    def at(offset, *shape):
        flat = torch.randn(5 * cols + 16, device="cuda", generator=g).to(dt)
        return flat, flat[offset:offset + 5 * cols].view(5, cols)
    _, h = at(1, 5, cols)
    _, y = at(2, 5, cols)
    whole, into = at(3, 5, cols)
    before = whole.clone()
    norm = torch.nn.RMSNorm(cols, eps=1e-6, device="cuda", dtype=dt).requires_grad_(False)
    norm.weight = torch.nn.Parameter(at(5, 5, cols)[1][0], requires_grad=False)
    q, s, n = V.add_rmsnorm_fp8(h, y, norm, out=into, return_norm=True)
    want = (h.float() + y.float()).to(dt)
    assert torch.equal(into, want)
    check(want, norm, q, s, n)
    whole[3:3 + 5 * cols] = before[3:3 + 5 * cols]
    assert torch.equal(whole, before)
    # the 8-bit output in an odd place, through the C entry point
    flat = torch.full((5 * cols + 16,), 7, device="cuda", dtype=torch.uint8)
    s2 = torch.empty(5, device="cuda")
    rc = V._lib.lib().verace_rmsnorm_fp8(want.data_ptr(), None, None, norm.weight.data_ptr(), 1e-6, 1, flat.data_ptr() + 3,
                                         s2.data_ptr(), None, 5, cols, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt],
                                         torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    # (against the formula: the order of a row's squares follows its words, and want starts at another place than h)
    check(want, norm, flat[3:3 + 5 * cols].clone().view(torch.float8_e4m3fn).view(5, cols), s2)
    assert (flat[:3] == 7).all() and (flat[3 + 5 * cols:] == 7).all()


def test_empty_and_refusals():
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    q, s = V.rmsnorm_fp8(torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16), norm)
    assert q.shape == (0, 64) and s.shape == (0,)
    x = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="match"):
        V.add_rmsnorm_fp8(x, x[:1], norm)
    with pytest.raises(AssertionError, match="contiguous"):
        V.add_rmsnorm_fp8(x, x, norm, out=torch.zeros(64, 2, device="cuda", dtype=torch.bfloat16).t())
    with pytest.raises(ValueError, match="inputs"):
        V.quantize_fp8(x.double())
    with pytest.raises(AssertionError):
        V.rmsnorm_fp8(x.float(), norm)
    with pytest.raises(RuntimeError, match="32768"):
        V.quantize_fp8(torch.zeros(1, 32769, device="cuda"))
    with pytest.raises(RuntimeError, match="32761"):
        V.quantize_fp8(torch.zeros(1, 32762, device="cuda"))
    with pytest.raises(RuntimeError, match="32761"):
        V.quantize_fp8(torch.zeros(32769, device="cuda")[1:].view(1, 32768))
    with pytest.raises(RuntimeError, match="no_grad"):
        V.quantize_fp8(x.clone().requires_grad_())
    with pytest.raises(AssertionError):
        V.quantize_fp8(torch.zeros(3, 0, device="cuda"))


def test_captured_and_on_another_stream():
    h, y, norm = data(33, 2048, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = V.add_rmsnorm_fp8(h, y, norm, out=torch.empty_like(h))
    torch.cuda.current_stream().wait_stream(side)
    into, hh = torch.empty_like(h), h.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = V.add_rmsnorm_fp8(hh, y, norm, out=into)
    hh.copy_(h)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cols", [5, 259, 1003, 5120])
def test_every_place_in_a_word(cols, dt):
    """h, y, the sum and the weights each start anywhere in a 16-byte word, with NaN before and behind them."""
    rows, word = 3, 16 // dt.itemsize
    h0, y0, norm0 = data(rows, cols, dt, 7)
    want = (h0.float() + y0.float()).to(dt)

    def at(t, off):
        base = torch.full((t.numel() + 2 * word,), math.nan, device="cuda", dtype=dt)
        view = base[off:off + t.numel()].view(t.shape)
        view.copy_(t)
        return base, view
    for i in range(word):
        for j, k in ((0, i), (i, 0), (3 * i % word, 5 * i % word), (i + 1 - i % 2 if i + 1 < word else 0, i)):
            (_, h), (_, y), (_, w) = at(h0, i), at(y0, j), at(norm0.weight.detach(), k)
            into, out = at(torch.zeros_like(h0), (i + j) % word)
            norm = torch.nn.RMSNorm(cols, eps=1e-6, device="cuda", dtype=dt)
            norm.weight = torch.nn.Parameter(w, requires_grad=False)
            assert norm.weight.data_ptr() == w.data_ptr()
            check(h0, norm0, *V.rmsnorm_fp8(h, norm))
            q, s, n = V.add_rmsnorm_fp8(h, y, norm, out=out, return_norm=True)
            assert torch.equal(out, want) and int(into.isnan().sum()) == 2 * word
            check(want, norm0, q, s, n)
