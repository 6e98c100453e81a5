"""int4_linear against the formula in 64 bits: sizes, groups, types, strides, special values.

Tolerances.  Each output is a sum of k products x (q - z) s with exact integers.  Summed in
fp32 in any order, every addition is off by at most 2^-23 of a partial sum of absolute terms
(truncating tensor-core additions included), so |y - ref| <= k 2^-23 sum |x w| + the output's
rounding (2^-8 |ref| bf16, 2^-11 fp16, 2^-24 fp32: half an ulp).  In the 2-norm, additions
inside a group make chains of at most 128 terms and the groups' sums are joined with rounded
additions: 4e-6 plus the output's rounding."""
import pytest
import torch

import verace_v1_b200 as V

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(m, n, k, group, dtype, zeros, bias, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    s = ((0.5 + torch.rand(groups, n, generator=g)) / k ** 0.5).to(dtype)
    z = torch.randint(0, 16, (groups, n), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    return x, q, s, z, b


def reference(x, q, s, z, b, group):
    n, k = q.shape[0], 2 * q.shape[1]
    codes = torch.empty(n, k, dtype=torch.float64)
    codes[:, 0::2], codes[:, 1::2] = (q & 15).double(), (q >> 4).double()
    of = torch.arange(k) // group
    w = (codes - (8.0 if z is None else z.double().t()[:, of])) * s.double().t()[:, of]
    y, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    return (y, size) if b is None else (y + b.double(), size + b.double().abs())


def check(y, ref, size, k, out_dtype):
    y, u = y.cpu().double(), HALF_ULP[out_dtype]
    assert torch.isfinite(y).all()
    bound = k * 2.0 ** -23 * size + u * ref.abs() + 1e-7 * (out_dtype == torch.float16)
    assert ((y - ref).abs() <= bound).all()
    assert (y - ref).norm() <= (u + 4e-6) * ref.norm() + 1e-7 * (out_dtype == torch.float16) * ref.numel() ** 0.5


def on_gpu(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 32, 32), (1, 3080, 1024, 128), (1, 17, 1056, 32), (2, 130, 96, 128), (3, 515, 4096, 64),
    (5, 33, 160, 64), (8, 256, 512, 32), (9, 31, 2080, 128), (16, 128, 1024, 64), (17, 100, 8192, 128),
    (24, 257, 544, 128), (31, 64, 64, 64), (33, 129, 1152, 32), (64, 384, 2048, 128), (65, 127, 768, 128),
    (150, 200, 320, 128), (7, 7, 16384, 128), (64, 260, 4128, 64)])
def test_matches_formula(m, n, k, group, dtype):
    for i, (zeros, bias) in enumerate([(False, False), (True, True)]):
        x, q, s, z, b = make(m, n, k, group, dtype, zeros, bias, seed=m * 1000 + n + k + i)
        ref, size = reference(x, q, s, z, b, group)
        xd, qd, sd, zd, bd = on_gpu(x, q, s, z, b)
        y = V.int4_linear(xd, qd, sd, zd, bd, group_size=group)
        assert y.shape == (m, n) and y.dtype == dtype
        check(y, ref, size, k, dtype)
        y32 = V.int4_linear(xd, qd, sd, zd, bd, group_size=group, out_dtype=torch.float32)
        assert y32.dtype == torch.float32
        check(y32, ref, size, k, torch.float32)
        assert torch.equal(y, V.int4_linear(xd, qd, sd, zd, bd, group_size=group)), "two calls differ"


@pytest.mark.parametrize("m,dtype", [(9, torch.bfloat16), (130, torch.float16), (20, torch.float32)])
def test_last_round_shares_its_inputs(m, dtype):
    """More row tiles than CTAs and few in the last round, with a long k."""
    n, k, group = 19400, 7200, 32 if m == 20 else 128
    x, q, s, z, b = make(m, n, k, group, dtype, True, True, seed=m)
    x[1, 7000], x[m - 1, 3] = 60000.0, -9000.0                     # far above the rest of their groups
    rows = torch.cat([torch.arange(0, n - 1600, 97), torch.arange(n - 1600, n)])
    ref, size = reference(x, q[rows], s[:, rows], z[:, rows], b[rows], group)
    y = V.int4_linear(*on_gpu(x, q, s, z, b), group_size=group, out_dtype=torch.float32)
    assert torch.isfinite(y).all()
    check(y[:, rows.cuda()], ref, size, k, torch.float32)


@pytest.mark.parametrize("m", [1, 6, 40])
def test_many_output_rows_and_long_inputs(m):
    """More rows than a wave of CTAs, and a long k for few rows (the split over k)."""
    for n, k, group in ((40001, 256, 128), (48, 65536, 128), (5, 32768, 32)):
        x, q, s, z, b = make(m, n, k, group, torch.bfloat16, True, False, seed=n + m)
        ref, size = reference(x, q, s, z, b, group)
        y = V.int4_linear(*on_gpu(x, q, s, z), group_size=group, out_dtype=torch.float32)
        check(y, ref, size, k, torch.float32)


@pytest.mark.parametrize("dtype,m", [(torch.bfloat16, 1), (torch.bfloat16, 7), (torch.bfloat16, 32), (torch.float16, 2),
                                     (torch.float16, 16), (torch.float32, 1), (torch.float32, 5), (torch.float32, 40)])
@pytest.mark.parametrize("n,k,group", [(300, 1024, 128), (9700, 512, 64), (130, 4096, 32)])
def test_inputs_of_weight_zero_add_nothing(n, k, group, dtype, m):
    """Codes equal to their zeros.  (Eight inputs a group: sums below 15 x 8 x 2^8 of the pieces, whose steps are
    2^-9, are exact.)"""
    x, q, s, z, b = make(m, n, k, group, dtype, True, False, seed=m + n + k)
    x[:, torch.arange(k) % group % (group // 8) != 1] = 0
    q[::2] = (z * 17).t().repeat_interleave(group // 2, 1)[::2]
    ref, size = reference(x, q, s, z, None, group)
    y = V.int4_linear(*on_gpu(x, q, s, z), group_size=group, out_dtype=torch.float32)
    assert (y[:, ::2] == 0).all()
    check(y, ref, size, k, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,group", [(1, 9700, 2304, 32), (3, 200, 16384, 128), (20, 300, 16384, 128), (20, 9700, 16384, 64),
                                         (40, 300, 16384, 64), (64, 200, 16384, 32)])
def test_sparse_inputs_count_once(m, n, k, group, dtype):
    """Few inputs that are not 0: in each group a large one and a small one, within eight inputs throughout
    every third run of 256, in the next eight throughout another third."""
    x, q, s, z, b = make(m, n, k, group, dtype, True, False, seed=m + n + k)
    x.zero_()
    for i in range(k // group):
        lo, run = i * group, i * group // 256
        if run % 3 < 2:
            x[:, lo + i % 8] = 1.0 + i % 5
            x[:, lo + (i + 1) % 8 + 8 * (run % 3)] = 1e-4
    if m > 2:
        x[1] = 0                                                   # a token of zeros beside the others
        x[2, group:] = 0
    rows = torch.arange(0, n, max(1, n // 200))
    ref, size = reference(x, q[rows], s[:, rows], z[:, rows], None, group)
    y = V.int4_linear(*on_gpu(x, q, s, z), group_size=group, out_dtype=torch.float32)
    check(y[:, rows.cuda()], ref, size, k, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,group", [(1, 300, 1024, 128), (9, 200, 4096, 64), (40, 130, 2048, 32)])
def test_inputs_at_the_ends_of_the_range(m, n, k, group, dtype):
    """Tokens near the largest and the smallest numbers of the type.  (Below the smallest normal number a
    product or a sum is off by half of 2^-149 more.)"""
    for e in (126, 119, 101, 98, -93, -110, -126, -130):
        x, q, s, z, b = make(m, n, k, group, dtype, True, False, seed=m + n + e)
        x = (x.double() * 2.0 ** e).clamp(-3.3e38, 3.3e38).to(dtype)
        ref, size = reference(x, q, s, z, None, group)
        y = V.int4_linear(*on_gpu(x, q, s, z), group_size=group, out_dtype=torch.float32).cpu().double()
        fits = size < 3e38
        assert fits.all() or e > 110
        bound = k * 2.0 ** -23 * size + 2.0 ** -24 * ref.abs() + k * 2.0 ** -149
        assert ((y - ref).abs() <= bound)[fits].all(), e
        if e == 126:                                               # few enough of them to fit
            x[:, 2:] = 0
            ref, size = reference(x, q, s, z, None, group)
            y = V.int4_linear(*on_gpu(x, q, s, z), group_size=group, out_dtype=torch.float32).cpu().double()
            assert (size < 3e38).sum() > size.numel() // 2
            assert ((y - ref).abs() <= k * 2.0 ** -23 * size)[size < 3e38].all()


# As stated in the header: y is the product with inputs each off by at most 2^-`bits` of its token's
# largest.
LOST = {torch.bfloat16: (32, 22, 21), torch.float16: (16, 26, 23), torch.float32: (1 << 20, 37, 37)}


def lost(x, q, s, z, group, m):
    most, few, many = LOST[x.dtype]
    _, weights = reference(torch.ones_like(x[:1]), q, s, z, None, group)         # sum |w|
    return 2.0 ** -(few if m <= most else many) * x.double().abs().amax(1, keepdim=True) * weights


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,group", [(1, 3080, 1024, 128), (7, 260, 4096, 64), (16, 200, 2048, 32), (24, 200, 2048, 128),
                                         (33, 130, 1024, 64), (64, 300, 1024, 32), (90, 260, 2048, 128)])
def test_groups_of_different_magnitude(m, n, k, group, dtype):
    """A group of ones above the others, and outputs whose weights are 0 there (which then adds exactly 0)."""
    x, q, s, z, b = make(m, n, k, group, dtype, True, False, seed=m + n + k)
    i = k // group // 2
    ones = slice(i * group, (i + 1) * group)
    q[::2, i * group // 2:(i + 1) * group // 2] = (z[i, ::2] * 17)[:, None]
    for below in (4, 10, 16, 22):
        xe = (x.float() * 2.0 ** -below).to(dtype)
        xe[:, ones] = 1
        ref, size = reference(xe, q, s, z, None, group)
        y = V.int4_linear(*on_gpu(xe, q, s, z), group_size=group, out_dtype=torch.float32).cpu().double()
        bound = k * 2.0 ** -23 * size + lost(xe, q, s, z, group, m)
        assert ((y - ref).abs() <= bound).all(), below


@pytest.mark.parametrize("m", [2, 16, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_inputs_far_below_the_rest_of_their_group(m, dtype):
    """Half of each group 2^14 above the other half, whose weights alone are not 0."""
    n, k, group = 200, 512, 64
    x, q, s, z, b = make(m, n, k, group, dtype, True, False, seed=m)
    low = torch.arange(k) % 2 == 1
    x = torch.where(low, (x.float() * 2.0 ** -8).to(dtype), (x.sign() * 64).to(dtype))
    q = (q & 0xF0) | z.t().repeat_interleave(group // 2, 1)        # code = zero at the even inputs
    ref, size = reference(x, q, s, z, None, group)
    y = V.int4_linear(*on_gpu(x, q, s, z), group_size=group, out_dtype=torch.float32).cpu().double()
    # the sums in the group run over q x and z X, in fp32: 2^-23 of up to twice 15 sum |x|, group terms
    sums = group * 2.0 ** -23 * 2 * 15 * (x.double().abs().view(m, -1, group).sum(2) @ s.double())
    assert ((y - ref).abs() <= k * 2.0 ** -23 * size + lost(x, q, s, z, group, m) + sums).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k,group", [(600, 300, 512, 128), (2050, 520, 288, 32), (513, 1160, 1024, 64)])
def test_prompt_sizes(m, n, k, group, dtype):
    x, q, s, z, b = make(m, n, k, group, dtype, True, True, seed=m)
    ref, size = reference(x, q, s, z, b, group)
    check(V.int4_linear(*on_gpu(x, q, s, z, b), group_size=group), ref, size, k, dtype)


def test_strides_shapes_and_streams():
    x, q, s, z, b = make(6, 96, 256, 64, torch.bfloat16, True, True, 1)
    ref, size = reference(x, q, s, z, b, 64)
    xd, qd, sd, zd, bd = on_gpu(x, q, s, z, b)
    wide = torch.full((6, 300), float("nan"), dtype=torch.bfloat16, device="cuda")
    for lo in (0, 8, 3):                     # aligned rows of a wider tensor, and rows at odd offsets
        wide[:, lo:lo + 256] = xd
        check(V.int4_linear(wide[:, lo:lo + 256], qd, sd, zd, bd, group_size=64), ref, size, 256, torch.bfloat16)
    check(V.int4_linear(xd.t().contiguous().t(), qd, sd, zd, bd, group_size=64), ref, size, 256, torch.bfloat16)
    y = V.int4_linear(xd.view(2, 3, 256), qd, sd, zd, bd, group_size=64)
    assert y.shape == (2, 3, 96)
    check(y.view(6, 96), ref, size, 256, torch.bfloat16)
    odd = torch.empty(q.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view_as(q)
    odd.copy_(qd)
    sn = torch.empty(2 * s.shape[0], s.shape[1], dtype=s.dtype, device="cuda")[::2]
    sn.copy_(sd)
    check(V.int4_linear(xd, odd, sn, zd, bd, group_size=64), ref, size, 256, torch.bfloat16)
    one = xd[:1].expand(6, 256)              # a broadcast row (stride 0)
    y = V.int4_linear(one, qd, sd, zd, bd, group_size=64)
    assert torch.equal(y, y[:1].expand(6, 96)) and torch.equal(y[0], V.int4_linear(xd, qd, sd, zd, bd, group_size=64)[0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = V.int4_linear(xd, qd, sd, zd, bd, group_size=64)
    st.synchronize()
    check(y, ref, size, 256, torch.bfloat16)


def test_empty_and_special_values():
    x, q, s, z, b = make(4, 40, 128, 32, torch.float32, True, False, 2)
    xd, qd, sd, zd = on_gpu(x, q, s, z)
    assert V.int4_linear(xd[:0], qd, sd, zd, group_size=32).shape == (0, 40)
    assert V.int4_linear(xd, qd[:0], sd[:, :0], zd[:, :0], group_size=32).shape == (4, 0)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        xi = x.to(dtype).clone()
        xi[1, 5], xi[2, 7], xi[3, 9] = float("inf"), float("nan"), -torch.finfo(dtype).max
        qi = q.clone()
        qi[:, 2] = 0xF0                      # k = 4: code 0, k = 5: code 15
        zi = torch.full_like(z, 7)
        y = V.int4_linear(*on_gpu(xi, qi, s.to(dtype), zi), group_size=32, out_dtype=torch.float32).cpu()
        assert (y[1] == float("inf")).all() and torch.isnan(y[2]).all() and torch.isfinite(y[0]).all()
        ref, size = reference(xi, qi, s.to(dtype), zi, None, 32)
        fits = ref[3].abs() < 1e38
        assert torch.isfinite(y[3][fits]).all()
        assert ((y[3] - ref[3]).abs()[fits] <= 128 * 2.0 ** -22 * size[3][fits]).all()


def test_quantized_module_and_graph():
    g = torch.Generator().manual_seed(3)
    lin = torch.nn.Linear(512, 200, bias=True)
    x = torch.randn(3, 512, generator=g).cuda().bfloat16()
    for symmetric in (True, False):
        mod = V.Int4Linear.from_linear(lin.cuda().bfloat16(), 64, symmetric)
        w = mod.dequantized()
        step = mod.scales.float().t().repeat_interleave(64, 1)
        # a code is off by half a step, by one bf16 rounding of the weight and of the scale; an
        # asymmetric zero is itself rounded by half a step
        assert ((w.float() - lin.weight.float()).abs() <= step * (0.51 if symmetric else 1.01) + 0.04 * step).all()
        ref = x.double() @ (w.double().t()) + lin.bias.double()
        with torch.no_grad():
            y = mod(x)
        # w is rounded to bf16 here (2^-8 each), the kernel's is not
        assert (y.double() - ref).norm() <= 2 ** -6 * ref.norm()
        graph = torch.cuda.CUDAGraph()
        out = mod(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = mod(x)
        graph.replay()
        assert torch.equal(out, y)
