"""process_logits and sample_logits against their formulas in 64 bits.

Tolerances.  process: at most five fp32 operations, each off by half an ulp of a value no
larger than |l| max(r, 1/r) + f c + p + |bias|: 6 * 2^-24 of that, plus the output's rounding.
sample: the token has to be the 64-bit formula's wherever that is clear of ties (its key ahead
of the next by 1e-4, the same token with either cut moved by 1e-5); a log-probability is z - max - log sum
with fp32 z, exp and log, each within a few 2^-24 of the sizes involved."""
import numpy as np
import pytest
import torch

import verace_v1_b200 as V

pytestmark = pytest.mark.gpu
INF = float("inf")
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------ process
def process_reference(l, tokens, lengths, prompts, r, p, f, ids, values, words):
    b, v = l.shape
    y, size = l.double().numpy().copy(), np.abs(l.double().numpy())
    for i in range(b):
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else max(0, min(int(lengths[i]), tokens.shape[1]))
            seen, count = set(), {}
            for j in range(n):
                t = int(tokens[i, j])
                if 0 <= t < v:
                    seen.add(t)
                    if j >= (0 if prompts is None else int(prompts[i])):
                        count[t] = count.get(t, 0) + 1
            for t in seen:
                y[i, t] = y[i, t] / r[i] if y[i, t] > 0 else y[i, t] * r[i]
                size[i, t] *= max(r[i], 1 / r[i])
            for t, c in count.items():
                y[i, t] -= f[i] * c + p[i]
                size[i, t] += abs(f[i]) * c + abs(p[i])
        if ids is not None:
            last = {int(t): float(x) for t, x in zip(ids[i], values[i]) if 0 <= int(t) < v}
            for t, x in last.items():
                y[i, t] += x
                size[i, t] += abs(x)
        if words is not None:
            w = words[i if words.shape[0] > 1 else 0].numpy().view(np.uint32)
            ok = (w[np.arange(v) // 32] >> (np.arange(v) % 32).astype(np.uint32)) & 1
            y[i, ok == 0] = -np.inf
    return torch.from_numpy(y), torch.from_numpy(size)


def check_process(out, ref, size, dtype):
    out = out.cpu().double()
    fine = torch.isfinite(ref)
    assert torch.equal(out[~fine], ref[~fine])
    tol = 6 * 2.0 ** -24 * size + HALF_ULP[dtype] * ref.abs() + 1e-7 * (dtype == torch.float16)
    assert ((out - ref).abs()[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,v,length", [(1, 1, 1), (1, 33, 5), (3, 1000, 64), (2, 4097, 300), (5, 32000, 1000),
                                        (2, 32001, 1), (64, 513, 37), (1, 163840, 20000), (40, 20011, 129),
                                        (9, 65600, 777), (300, 96, 40)])
def test_process_matches_formula(b, v, length, dtype):
    g = torch.Generator().manual_seed(b * 7 + v + length)
    l = (3 * torch.randn(b, v, generator=g)).to(dtype)
    tokens = torch.randint(-2, v + 2, (b, length), generator=g)
    tokens[:, ::3] = tokens[:, :1].clone()                       # one token many times
    lengths = torch.randint(0, length + 1, (b,), generator=g)
    prompts = torch.randint(0, length + 1, (b,), generator=g)
    lengths[0], prompts[0] = length, length // 2
    if b > 1:
        lengths[1], prompts[1] = 0, 0
    if b > 2:
        lengths[2], prompts[2] = length + 9, -4
    r, p, f = 1 + torch.rand(b, generator=g), torch.rand(b, generator=g), 0.3 * torch.rand(b, generator=g) - 0.1
    n = min(v, 20)
    ids = torch.stack([torch.randperm(v, generator=g)[:n] for _ in range(b)])
    ids[:, -1] = -1
    values = 5 * torch.randn(b, n, generator=g)
    words = torch.randint(-2 ** 31, 2 ** 31, (b, (v + 31) // 32), generator=g).int()
    if b > 1:
        words[1] = 0                                     # nothing left
    for kw in ({}, {"bias": 1}, {"mask": 1}, {"bias": 1, "mask": 1, "i32": 1}, {"out32": 1, "mask": 1}):
        i = ids if kw.get("bias") else None
        x = values if kw.get("bias") else None
        w = words if kw.get("mask") else None
        cast = (lambda t: t.int()) if kw.get("i32") else (lambda t: t)
        ref, size = process_reference(l, tokens, lengths, prompts, r.double().numpy(), p.double().numpy(),
                                      f.double().numpy(), i, x, w)
        odt = torch.float32 if kw.get("out32") else dtype
        out = V.process_logits(l.cuda(), cast(tokens).cuda(), cast(lengths).cuda(), cast(prompts).cuda(),
                               repetition_penalty=r.cuda(), presence_penalty=p.cuda(), frequency_penalty=f.cuda(),
                               bias_ids=None if i is None else cast(i).cuda(), bias_values=None if x is None else x.cuda(),
                               allowed=None if w is None else w.cuda(), out_dtype=odt)
        assert out.dtype == odt
        check_process(out, ref, size, odt)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,v,length,among,n,pad", [(130, 32776, 601, 32776, 40, 0), (65, 65543, 4000, 6000, 20, 1),
                                                    (66, 65600, 50, 65600, 700, 8), (130, 32800, 0, 1, 900, 0)])
def test_process_many_wide_rows(b, v, length, among, n, pad, dtype):
    """Histories over few or many tokens, biases few or many, of one token or many, in place too."""
    g = torch.Generator().manual_seed(b + v + length)
    l = (3 * torch.randn(b, v + pad, generator=g)).to(dtype)[:, :v]
    tokens = torch.randint(-3, among, (b, max(length, 1)), generator=g)[:, :length]
    lengths, prompts = torch.randint(0, length + 1, (b,), generator=g), torch.randint(0, length + 1, (b,), generator=g)
    lengths[:3], prompts[:2] = length, torch.tensor([0, length])
    r, p, f = 1 + torch.rand(b, generator=g), torch.rand(b, generator=g), 0.3 * torch.rand(b, generator=g) - 0.1
    ids = torch.randint(-1, min(v, 20000), (b, n), generator=g)
    ids[1] = 7                                                   # one token, all its biases
    values = 5 * torch.randn(b, n, generator=g)
    words = torch.randint(-2 ** 31, 2 ** 31, (b, (v + 31) // 32), generator=g).int()
    words[2] = 0
    ref, size = process_reference(l, tokens, lengths, prompts, r.double().numpy(), p.double().numpy(),
                                  f.double().numpy(), ids, values, words)
    for i32, odt, place in ((False, torch.float32, False), (True, dtype, False), (False, dtype, True)):
        cast = (lambda t: t.int()) if i32 else (lambda t: t)
        ld = torch.empty(b, v + pad, dtype=dtype, device="cuda")[:, :v].copy_(l)
        out = V.process_logits(ld, cast(tokens).cuda(), lengths.cuda(), prompts.cuda(), repetition_penalty=r.cuda(),
                               presence_penalty=p.cuda(), frequency_penalty=f.cuda(), bias_ids=cast(ids).cuda(),
                               bias_values=values.cuda(), allowed=words.cuda(), out_dtype=odt, out=ld if place else None)
        assert not place or out.data_ptr() == ld.data_ptr()
        check_process(out, ref, size, odt)


@pytest.mark.parametrize("b,v,length", [(2, 3000, 900), (130, 32776, 300), (1, 400, (1 << 20) + 5), (2, 5000, 20000)])
def test_process_repetition_penalty_is_rounded_once(b, v, length):
    """l / r and l r themselves, not a product with a rounded 1 / r: equal to the last bit, tiny r included."""
    g = torch.Generator().manual_seed(v)
    tokens = torch.randint(0, v, (b, length), generator=g)
    r = 1 + torch.rand(b, generator=g)
    r[0] = 2e-39                                                   # (its reciprocal is beyond fp32)
    seen = torch.zeros(b, v, dtype=torch.bool).scatter_(1, tokens, True)
    for dtype in (torch.float32, torch.bfloat16):
        l = torch.randn(b, v, generator=g).to(dtype)
        l[0] = (l[0].float() * 1e-3).to(dtype)
        x = l.float()
        want = torch.where(seen, torch.where(x > 0, x / r[:, None], x * r[:, None]), x)
        out = V.process_logits(l.cuda(), tokens.cuda(), None, torch.full((b,), length).cuda(), repetition_penalty=r.cuda(),
                               out_dtype=torch.float32)
        assert torch.isfinite(want).all() and torch.equal(out.cpu(), want)


def test_process_lengths_beyond_32_bits():
    g = torch.Generator().manual_seed(21)
    l, tokens = torch.randn(3, 500, generator=g).cuda(), torch.randint(0, 500, (3, 60), generator=g).cuda()
    kw = dict(repetition_penalty=1.5, presence_penalty=0.5)
    for big in (1 << 31, (1 << 32) + 1, (1 << 63) - 1):
        big = torch.full((3,), big, device="cuda")
        assert torch.equal(V.process_logits(l, tokens, big, **kw), V.process_logits(l, tokens, **kw))
        want = V.process_logits(l, tokens, repetition_penalty=1.5)       # all of it the prompt
        assert not torch.equal(want, l)
        assert torch.equal(V.process_logits(l, tokens, None, big, **kw), want)
        want = V.process_logits(l, tokens, repetition_penalty=1.5, presence_penalty=0.5)
        assert torch.equal(V.process_logits(l, tokens, None, -big, **kw), want)


def test_process_parts_alone_and_scalars():
    g = torch.Generator().manual_seed(5)
    l = torch.randn(4, 700, generator=g)
    tokens = torch.randint(0, 700, (4, 50), generator=g)
    ld, td = l.cuda(), tokens.cuda()
    assert torch.equal(V.process_logits(ld), ld)                       # nothing asked: the same values
    assert torch.equal(V.process_logits(ld, td), ld)                   # neutral penalties
    ones = np.ones(4)
    ref, size = process_reference(l, tokens, None, None, 1.5 * ones, 0.25 * ones, 0.5 * ones, None, None, None)
    check_process(V.process_logits(ld, td, repetition_penalty=1.5, presence_penalty=0.25, frequency_penalty=0.5),
                  ref, size, torch.float32)
    word = torch.randint(-2 ** 31, 2 ** 31, (1, 22), generator=g).int()   # one mask for every row
    ref, size = process_reference(l, None, None, None, ones, ones, ones, None, None, word)
    check_process(V.process_logits(ld, allowed=word.cuda()), ref, size, torch.float32)
    empty = torch.empty(4, 0, dtype=torch.long, device="cuda")
    assert torch.equal(V.process_logits(ld, empty, repetition_penalty=2.0, bias_ids=empty,
                                        bias_values=empty.float()), ld)
    assert V.process_logits(ld[:0], td[:0]).shape == (0, 700) and V.process_logits(ld[:, :0]).shape == (4, 0)


@pytest.mark.parametrize("v", [50000, 262144, 500000, 900001])
def test_process_large_vocabularies(v):
    g = torch.Generator().manual_seed(v)
    l = torch.randn(2, v, generator=g)
    tokens = torch.randint(0, v, (2, 3000), generator=g)
    tokens[:, 500:900] = v - 1
    ids = torch.randint(0, v, (2, 40), generator=g)
    values = torch.randn(2, 40, generator=g)
    ones = np.ones(2)
    ref, size = process_reference(l, tokens, None, torch.tensor([100, 2000]), 1.7 * ones, 0.3 * ones, 0.01 * ones, ids,
                                  values, None)
    out = V.process_logits(l.cuda(), tokens.cuda(), None, torch.tensor([100, 2000]).cuda(), repetition_penalty=1.7,
                           presence_penalty=0.3, frequency_penalty=0.01, bias_ids=ids.cuda(), bias_values=values.cuda())
    check_process(out, ref, size, torch.float32)


def test_process_very_long_history():
    """A history beyond the 20 bits of a counter."""
    n = (1 << 20) + 77
    tokens = torch.full((1, n), 5)
    tokens[0, ::3] = 100
    l = torch.zeros(1, 300)
    ref, size = process_reference(l, tokens, None, torch.tensor([3]), np.ones(1), 0.25 * np.ones(1),
                                  2.0 ** -10 * np.ones(1), torch.tensor([[5, 7]]), torch.tensor([[1.0, 2.0]]), None)
    out = V.process_logits(l.cuda(), tokens.cuda(), None, torch.tensor([3]).cuda(), presence_penalty=0.25,
                           frequency_penalty=2.0 ** -10, bias_ids=torch.tensor([[5, 7]]).cuda(),
                           bias_values=torch.tensor([[1.0, 2.0]]).cuda())
    check_process(out, ref, size, torch.float32)


def test_process_many_biases():
    """More biases in one CTA's range than it lists, with repeats."""
    g = torch.Generator().manual_seed(11)
    l = torch.randn(2, 3000, generator=g)
    ids = torch.randint(0, 2000, (2, 2500), generator=g)
    values = torch.randn(2, 2500, generator=g)
    ones = np.ones(2)
    ref, size = process_reference(l, None, None, None, ones, ones, ones, ids, values, None)
    check_process(V.process_logits(l.cuda(), bias_ids=ids.cuda(), bias_values=values.cuda()), ref, size, torch.float32)


def test_process_equal_bias_ids_the_last_holds():
    l = torch.zeros(2, 64, device="cuda")
    ids = torch.tensor([[3, 5, 3, 3], [7, 7, 8, -1]], device="cuda")
    values = torch.tensor([[1.0, 2.0, 4.0, 8.0], [1.0, -3.0, 5.0, 9.0]], device="cuda")
    out = V.process_logits(l, bias_ids=ids, bias_values=values).cpu()
    assert out[0, 3] == 8 and out[0, 5] == 2 and out[1, 7] == -3 and out[1, 8] == 5 and out.abs().sum() == 18


@pytest.mark.parametrize("dtype", TYPES)
def test_process_special_values(dtype):
    v = 70
    l = torch.zeros(1, v)
    l[0, :6] = torch.tensor([float("nan"), INF, -INF, float("nan"), torch.finfo(dtype).min, torch.finfo(dtype).max])
    l[0, 6] = -0.0
    l = l.to(dtype).cuda()
    words = torch.full((1, 3), -1, dtype=torch.int32)
    words[0, 0] = ~1                                                   # token 0 (a NaN) is masked
    tokens = torch.tensor([[1, 2, 3, 6, 20]], device="cuda")
    out = V.process_logits(l, tokens, repetition_penalty=2.0, allowed=words.cuda()).cpu().float()[0]
    assert out[0] == -INF and out[1] == INF and out[2] == -INF and torch.isnan(out[3])
    assert out[4] == torch.finfo(dtype).min and out[5] == torch.finfo(dtype).max
    assert (out[6:] == 0).all()
    low = torch.full((1, 1), torch.finfo(torch.float32).min, device="cuda")   # an additive mask's lowest value
    out = V.process_logits(l, bias_ids=torch.tensor([[20]], device="cuda"), bias_values=low).cpu().float()[0, 20]
    assert out == (torch.finfo(torch.float32).min if dtype == torch.float32 else -INF)


def test_process_strides_in_place_and_streams():
    g = torch.Generator().manual_seed(6)
    l = torch.randn(3, 900, generator=g)
    tokens = torch.randint(0, 900, (3, 80), generator=g)
    ones = np.ones(3)
    ref, size = process_reference(l, tokens, None, None, 1.3 * ones, 0.5 * ones, 0.1 * ones, None, None, None)
    kw = dict(repetition_penalty=1.3, presence_penalty=0.5, frequency_penalty=0.1)
    for dtype in TYPES:
        ref, size = process_reference(l.to(dtype), tokens, None, None, 1.3 * ones, 0.5 * ones, 0.1 * ones, None, None,
                                      None)
        for lo, ld in ((0, 912), (1, 903), (4, 928)):
            wide = torch.zeros(3, ld, dtype=dtype, device="cuda")
            wide[:, lo:lo + 900] = l.to(dtype).cuda()
            view = wide[:, lo:lo + 900]
            tw = torch.zeros(3, 101, dtype=torch.long, device="cuda")
            tw[:, 7:87] = tokens.cuda()
            check_process(V.process_logits(view, tw[:, 7:87], **kw), ref, size, dtype)
            check_process(V.process_logits(view, tokens.t().contiguous().t().cuda(), **kw), ref, size, dtype)
            before = wide.clone()
            assert V.process_logits(view, tw[:, 7:87], out=view, **kw) is view
            check_process(view, ref, size, dtype)
            assert torch.equal(wide[:, :lo], before[:, :lo]) and torch.equal(wide[:, lo + 900:], before[:, lo + 900:])
    st = torch.cuda.Stream()
    ld, td = l.cuda(), tokens.cuda()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        out = V.process_logits(ld, td, **kw)
    st.synchronize()
    ref, size = process_reference(l, tokens, None, None, 1.3 * ones, 0.5 * ones, 0.1 * ones, None, None, None)
    check_process(out, ref, size, torch.float32)


# ------------------------------------------------------------------ sample
def sample_reference(l, noise, t, k, p, minp):
    """(token, logprob, clear) of one row in 64 bits; clear: the same token with the cuts by mass
    and by min_p moved by 1e-5 either way, and its key ahead of the next by 1e-4."""
    l = np.where(np.isnan(l), -np.inf, l)
    z = l / t if t > 0 else l
    top = z.max()
    if top == -np.inf:
        return -1, -np.inf, True
    if top == np.inf:                                            # the infinities share the mass
        z, top = np.where(z == top, 0.0, -np.inf), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(z == top, 1.0, np.exp(z - top))
    chosen, clear = [], True
    for eps in (0.0, 1e-5, -1e-5):
        keep = z > -np.inf
        key = z
        if t > 0:
            if 0 < k < len(z):
                keep &= z >= np.sort(z)[::-1][k - 1]
            if p < 1:
                values, at = np.unique(z[keep], return_inverse=True)
                masses = np.bincount(at, weights=w[keep])[::-1]              # by value, descending
                above = np.concatenate([[0.0], np.cumsum(masses)[:-1]])
                inside = above < p * masses.sum() * (1 + eps)
                inside[0] = True
                keep &= z >= values[::-1][inside].min()
            keep &= (w >= minp * (1 + eps)) | (z == top)
            key = np.where(keep, z - np.log(noise), -np.inf)
        chosen.append(int(np.argmax(key)))
        if t > 0:
            others = np.delete(key, chosen[-1])
            clear &= len(others) == 0 or not (key[chosen[-1]] - others.max() < 1e-4)
    token = chosen[0]
    return token, (0.0 if z[token] == top else z[token] - top) - np.log(w.sum()), clear and len(set(chosen)) == 1


def check_sample(l, noise, t, k, p, minp, most_clear=True, **kw):
    b, v = l.shape
    args = [x if isinstance(x, torch.Tensor) else torch.full((b,), float(x)) for x in (t, k, p, minp)]
    tok, lp = V.sample_logits(l.cuda(), None if noise is None else noise.cuda(),
                              temperature=t.cuda() if isinstance(t, torch.Tensor) else t,
                              top_k=k.cuda() if isinstance(k, torch.Tensor) else k,
                              top_p=p.cuda() if isinstance(p, torch.Tensor) else p,
                              min_p=minp.cuda() if isinstance(minp, torch.Tensor) else minp)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (b,)
    tok, lp, clears = tok.cpu(), lp.cpu(), 0
    ln = l.double().numpy()
    nn = None if noise is None else noise.double().numpy()
    for i in range(b):
        ti = float(args[0][i])
        token, ref, clear = sample_reference(ln[i], None if nn is None else nn[i], ti, int(args[1][i]),
                                             float(args[2][i]), float(args[3][i]))
        if not clear:
            continue
        clears += 1
        assert int(tok[i]) == token, (i, int(tok[i]), token)
        if ref == -np.inf:
            assert lp[i] == -INF
        else:
            size = np.abs(np.where(np.isfinite(ln[i]), ln[i], 0)).max() / (ti or 1)
            assert abs(float(lp[i]) - ref) <= 2.0 ** -21 * (2 + 2 * size + abs(ref))
    assert clears >= 0.8 * b or not most_clear
    return tok, lp


def draw(b, v, seed, masked=0.0, dtype=torch.float32, std=2.5):
    g = torch.Generator().manual_seed(seed)
    l = std * torch.randn(b, v, generator=g)
    if masked:
        l[torch.rand(b, v, generator=g) < masked] = -INF
    return l.to(dtype), torch.empty(b, v).exponential_(generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,v", [(1, 1), (2, 3), (5, 31), (3, 1000), (4, 4099), (2, 32000), (7, 32001), (1, 163840),
                                 (40, 20011), (300, 130)])
def test_sample_matches_formula(b, v, dtype):
    for seed, (t, k, p, minp, masked) in enumerate([
            (0.0, 0, 1.0, 0.0, 0.0), (1.0, 0, 1.0, 0.0, 0.0), (0.7, 50, 1.0, 0.0, 0.3), (1.3, 0, 0.9, 0.0, 0.0),
            (1.0, 1, 1.0, 0.0, 0.0), (0.8, 40, 0.6, 0.05, 0.5), (1.0, 0, 1.0, 0.1, 0.9), (1.0, 1000, 0.5, 0.0, 0.0)]):
        l, noise = draw(b, v, 100 * seed + b + v, masked, dtype)
        check_sample(l, noise if t else None, t, k, p, minp, most_clear=b * v > 100)


@pytest.mark.parametrize("v,dtype", [(20501, torch.float32), (20608, torch.float32), (41001, torch.bfloat16)])
def test_sample_many_rows_too_long_to_hold(v, dtype):
    """More rows than shared memory holds, values of every kind at the rows' ends among them."""
    b = 300
    l, noise = draw(b, v, 11, dtype=dtype)
    lowest = torch.finfo(dtype).min
    l[1], l[2], l[3, 100:], l[6], l[7] = -INF, -INF, -INF, 0.0, lowest
    l[2, v - 1] = lowest
    l[4, ::7] = float("nan")
    l[5, 5:9], l[8, v - 1], l[b - 1] = INF, 30.0, lowest
    for t, k, p, minp in ((0.8, 50, 0.9, 0.0), (1.3, 0, 0.7, 0.0), (1.0, 5000, 1.0, 0.0), (0.7, 0, 1.0, 0.01),
                          (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)):
        check_sample(l, noise if t else None, t, k, p, minp)


def test_sample_per_row_controls():
    b, v = 24, 5000
    l, noise = draw(b, v, 1, 0.2)
    g = torch.Generator().manual_seed(2)
    t = torch.rand(b, generator=g) * 2
    t[::5] = 0
    k = torch.randint(0, 60, (b,), generator=g)
    p = torch.rand(b, generator=g) * 1.2
    minp = torch.rand(b, generator=g) * 0.1
    l[3] = -INF
    l[4] = float("nan")
    check_sample(l, noise, t, k, p, minp)


def test_sample_ties_and_extremes():
    v = 300
    flat = torch.zeros(4, v)
    noise = torch.empty(4, v).exponential_(generator=torch.Generator().manual_seed(3))
    tok, lp = V.sample_logits(flat.cuda(), temperature=0)
    assert (tok == 0).all() and torch.allclose(lp.cpu(), torch.full((4,), -float(np.log(v))), rtol=1e-6)
    # k = 5 over equal values keeps them all: the draw is the smallest noise
    tok, _ = V.sample_logits(flat.cuda(), noise.cuda(), top_k=5)
    assert torch.equal(tok.cpu(), noise.argmin(1))
    tok, _ = V.sample_logits(flat.cuda(), noise.cuda(), top_p=0.1)
    assert torch.equal(tok.cpu(), noise.argmin(1))
    zeros = flat.clone()
    zeros[:, ::2] = -0.0                                               # -0 and 0 are one value
    tok, _ = V.sample_logits(zeros.cuda(), noise.cuda(), top_k=1)
    assert torch.equal(tok.cpu(), noise.argmin(1))
    tok, _ = V.sample_logits(flat.cuda(), torch.ones(4, v).cuda())     # equal keys: the lowest index
    assert (tok == 0).all()
    l, noise = draw(3, v, 4)
    l[0, 17], l[1, 5], l[1, 250] = INF, INF, INF
    l[2] = -INF
    l[2, 299] = torch.finfo(torch.float32).min
    for kw in ({"temperature": 0.0}, {"temperature": 1.0}, {"temperature": 0.5, "top_p": 0.5}, {"top_k": 1}):
        tok, lp = V.sample_logits(l.cuda(), noise.cuda(), **kw)
        tok, lp = tok.cpu(), lp.cpu()
        assert tok[0] == 17 and tok[1] in (5, 250) and tok[2] == 299
        assert lp[0] == 0 and abs(lp[1] + np.log(2)) < 1e-6 and lp[2] == 0
    # top_p = 0 keeps the largest; a temperature that sends z out of range still chooses it
    l, noise = draw(6, 1000, 5)
    for kw in ({"top_p": 0.0}, {"min_p": 1.0}, {"temperature": 1e-30}):
        tok, _ = V.sample_logits(l.cuda(), noise.cuda(), **kw)
        if "temperature" not in kw:
            assert torch.equal(tok.cpu(), l.argmax(1))
        else:
            assert (l.gather(1, tok.cpu()[:, None]) > 0).all()
    peaked = torch.full((1, 1000), -12.0)
    peaked[0, 3] = 3.0                                                 # log p near 0 keeps its digits
    _, lp = V.sample_logits(peaked.cuda(), temperature=0)
    assert abs(float(lp) / -np.log1p(999 * np.exp(-15.0)) - 1) < 1e-5
    assert V.sample_logits(l[:0].cuda(), temperature=0)[0].shape == (0,)


@pytest.mark.parametrize("b,v", [(40, 3000), (300, 20608), (2, 1100000)])
@pytest.mark.parametrize("offset", [-6e4, 300.0, 2e5, -3e7])
def test_sample_logits_far_from_zero(b, v, offset):
    """z is against the row's largest: what all of a row's logits have in common costs no digits of the noise."""
    l, noise = draw(b, v, v)
    l = l + offset
    for t, k, p, minp in ((0.7, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.8, 0.01), (1.3, 0, 1.0, 0.05)):
        check_sample(l, noise, t, k, p, minp, most_clear=b < 300 and v < 1000000)


@pytest.mark.parametrize("kw", [{}, {"top_k": 3000}, {"top_p": 0.9999}, {"min_p": 1e-30}])
@pytest.mark.parametrize("b,v", [(2, 3000), (300, 20608)])
def test_sample_subnormal_noise(b, v, kw):
    """-log(noise) of subnormal noise (88 to 103) beside the smallest normal numbers', and of 0 (infinite)."""
    g = torch.Generator().manual_seed(v)
    l = 0.1 * torch.randn(b, v, generator=g)
    noise = 1.2e-38 * (1 + torch.rand(b, v, generator=g))
    noise[:, ::50] = 2.0 ** -149 * torch.randint(1, 1 << 22, noise[:, ::50].shape, generator=g)
    l[:, 77], noise[:, 77] = 20.0, 0.5                           # kept, but far from chosen
    l[1, ::50] -= 30.0                                           # the normal ones win over the subnormal
    tok, _ = V.sample_logits(l.cuda(), noise.cuda(), **kw)
    score = l.double() - noise.double().log()
    if kw.get("top_k", v) < v:
        score[l < l.sort(dim=1, descending=True).values[:, kw["top_k"] - 1:kw["top_k"]]] = -INF
    if "min_p" in kw:
        score[l.double() - l.max(1, keepdim=True).values < np.log(1e-30)] = -INF
    if "top_p" in kw:
        score[:, :77], score[:, 78:] = -INF, -INF                # (all but e^-20 of the mass)
    best = score.max(1).values
    assert (best - score.gather(1, tok.cpu()[:, None])[:, 0] <= 1e-4).all()
    noise[0, 1234], l[0, 1234] = 0.0, -10.0
    if not kw:
        assert int(V.sample_logits(l.cuda(), noise.cuda())[0][0]) == 1234


@pytest.mark.parametrize("b,v", [(3, 1000), (300, 20608), (2, 1100000)])
def test_sample_infinite_temperatures(b, v):
    """Rows of infinite T draw evenly from what is not masked: the smallest noise, log p = -log of its count."""
    l, noise = draw(b, v, v, 0.3)
    l[1] = -INF
    l[1, 5:9] = 3e38
    t = torch.ones(b)
    t[:2] = INF
    for kw in ({}, {"top_k": 20}, {"top_p": 0.5}):
        tok, lp = V.sample_logits(l.cuda(), noise.cuda(), temperature=t.cuda(), **kw)
        for i in range(2):
            there = l[i] > -INF
            if kw:                                                     # (the logits' order, with equal masses)
                there &= l[i] >= l[i].sort(descending=True).values[19 if "top_k" in kw else (int(there.sum()) - 1) // 2]
            assert int(tok[i]) == int(torch.where(there, noise[i], INF).argmin())
            assert abs(float(lp[i]) + np.log(int((l[i] > -INF).sum()))) <= 1e-5


def test_sample_top_k_beyond_32_bits():
    l, noise = draw(4, 3000, 12)
    want = V.sample_logits(l.cuda(), noise.cuda())
    assert not torch.equal(want[0].cpu(), l.argmax(1))
    for k in (1 << 31, (1 << 32) + 1, (1 << 63) - 1, -(1 << 40) + 1):
        for top_k in (k, torch.full((4,), k, device="cuda")):
            got = V.sample_logits(l.cuda(), noise.cuda(), top_k=top_k)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_sample_draws_follow_the_softmax():
    l = torch.tensor([2.0, 1.0, 0.0, -1.0, 3.0, -INF, 0.5, 2.5])
    n = 20000
    noise = torch.empty(n, 8).exponential_(generator=torch.Generator().manual_seed(7)).cuda()
    for kw, keep in (({}, torch.tensor([1, 1, 1, 1, 1, 0, 1, 1.])), ({"top_k": 3}, torch.tensor([1, 0, 0, 0, 1, 0, 0, 1.]))):
        tok, _ = V.sample_logits(l.expand(n, 8).cuda(), noise, **kw)
        prob = torch.softmax(l, 0) * keep
        prob = prob / prob.sum()
        freq = torch.bincount(tok.cpu(), minlength=8).double() / n
        # six standard deviations of a count
        assert ((freq - prob).abs() <= 6 * (prob * (1 - prob) / n).sqrt()).all()


def test_sample_vocabularies_of_any_size():
    """Rows for one CTA, for clusters of up to sixteen, and beyond what a cluster holds."""
    for b, v, dtype in ((200, 20000, torch.float32), (3, 262144, torch.bfloat16), (2, 400001, torch.float32),
                        (2, 800003, torch.float32)):
        l, noise = draw(b, v, v, 0.1, dtype)
        check_sample(l, noise, 1.0, 0, 0.95, 0.0)
        check_sample(l, noise, 0.7, 200, 0.8, 0.001)
        check_sample(l, noise, 1.5, 0, 1.0, 0.0)
        check_sample(l, None, 0.0, 0, 1.0, 0.0)


def test_sample_masses_of_very_long_rows():
    """2^24 equal values at the top: their mass alone is 2^64 of the units that shorter rows have."""
    v, n = (1 << 24) + (1 << 22), 1 << 24
    l = torch.zeros(1, v, device="cuda")
    l[:, n:] = -1.0
    noise = torch.ones(1, v, device="cuda")
    noise[0, 5], noise[0, v - 9] = 0.5, 1e-6
    for kw, token in (({"top_p": 0.5}, 5), ({"top_p": 0.999}, v - 9), ({}, v - 9), ({"top_k": 7}, 5)):
        tok, lp = V.sample_logits(l, noise, **kw)
        assert int(tok) == token
        want = (0.0 if token == 5 else -1.0) - np.log(n + (v - n) * np.exp(-1.0))
        # (4096 fp32 additions a thread, of a tenth of the sum)
        assert abs(float(lp) - want) <= 4096 * 2.0 ** -24 * 0.1 + 2.0 ** -21 * 20


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_cuts_among_many_equal_values(dtype):
    """Few distinct values, values around zero and of every size: the cut falls into crowded bins."""
    g = torch.Generator().manual_seed(9)
    v = 30000
    rows = [torch.randint(0, 6, (v,), generator=g).float(), torch.randn(v, generator=g) * 1e-4,
            10.0 ** (torch.rand(v, generator=g) * 8 - 6) * torch.randn(v, generator=g).sign(),
            torch.randn(v, generator=g) * 200, torch.full((v,), 1.5), 100 + torch.rand(v, generator=g) * 1e-3,
            torch.randint(0, 2, (v,), generator=g).float() * 1e4]
    l = torch.stack(rows).to(dtype)
    noise = torch.empty(l.shape).exponential_(generator=g)
    for t, k, p, minp in ((1.0, 1000, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 7, 0.5, 0.0), (50.0, 20000, 0.9, 0.0),
                          (0.01, 100, 0.7, 0.0)):
        check_sample(l, noise, t, k, p, minp, most_clear=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b", [1, 64])
def test_sample_rows_crowded_at_one_end(b, dtype):
    """Rows whose kept tokens lie in one CTA's part, by more than it lists, and not in the others'."""
    v = 163840
    l, noise = draw(b, v, 31 + b, dtype=dtype)
    block = torch.full((b, v), -INF, dtype=dtype)                # a block of tokens allowed, all equal
    for lo in (0, 60000, v - 20000):
        block.fill_(-INF)
        block[:, lo:lo + 20000] = 0.0
        check_sample(block, noise, 1.0, 50, 1.0, 0.0)
        block[:, lo:lo + 20000] = l[:, lo:lo + 20000]            # and not equal
        check_sample(block, noise, 1.0, 1000, 0.9, 0.0)
    ties = l.clone()
    ties[:, :10000] = 14.0                                       # equal ones at the top, in front of the rest
    check_sample(ties, noise, 1.0, 50, 1.0, 0.0)
    check_sample(ties, noise, 1.0, 50, 0.9, 0.0)
    ties[:, :v // 2] = 14.0
    check_sample(ties, noise, 1.0, 1000, 1.0, 0.01)
    check_sample(ties, noise, 1.0, 0, 0.3, 0.0)
    padded = (0.1 * l.float()).to(dtype)                         # nearly flat, the vocabulary's end padded
    padded[:, 150000:] = -INF
    check_sample(padded, noise, 20.0, 50, 1.0, 0.0)
    check_sample(padded, noise, 20.0, 50, 0.8, 0.01)
    check_sample(l, noise, 1.0, 32000, 0.95, 0.0)                # lists of about what a CTA holds
    check_sample(l, noise, 1.0, 32000, 1.0, 0.0)


def test_sample_strides_and_streams():
    l, noise = draw(5, 777, 8, 0.1)
    lw, nw = torch.zeros(5, 800, device="cuda"), torch.ones(5, 779, device="cuda")
    lw[:, 3:780], nw[:, 1:778] = l.cuda(), noise.cuda()
    kw = dict(temperature=0.9, top_k=30, top_p=0.8, min_p=0.01)
    want = V.sample_logits(l.cuda(), noise.cuda(), **kw)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = V.sample_logits(lw[:, 3:780], nw[:, 1:778], **kw)
    st.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    got = V.sample_logits(l.t().contiguous().t().cuda(), noise.cuda(), **kw)
    assert torch.equal(want[0], got[0])
    check_sample(l, noise, 0.9, 30, 0.8, 0.01)
