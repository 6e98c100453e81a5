"""CPU checks of the 4-bit products, logits processing and token choice: the quantiser, and what
the entry points refuse (placeholder pointers only where no GPU is visible)."""
import ctypes

import pytest
import torch

import verace_v1_b200 as V
from verace_v1_b200 import _lib

host_only = pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers: run without a GPU only")
FAKE = ctypes.c_void_p(256)


def _err():
    return _lib.lib().verace_last_error().decode()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,group", [(32, 32), (96, 64), (256, 128), (160, 128)])
@pytest.mark.parametrize("symmetric", [True, False])
def test_quantised_weights_are_within_a_step(dtype, k, group, symmetric):
    g = torch.Generator().manual_seed(k + group)
    w = torch.randn(9, k, generator=g).to(dtype)
    w[2] = 0
    w[3] = w[3].abs()
    q, s, z = V.quantize_int4(w, group, symmetric)
    assert q.shape == (9, k // 2) and s.shape == (-(-k // group), 9) and s.dtype == dtype
    assert (z is None) == symmetric
    back = V.dequantize_int4(q, s, z, group_size=group).double()
    step = s.double().t()[:, torch.arange(k) // group]
    # half a step by the code; a clamped end loses what rounding the scale shrank (16 half-ulps
    # of the dtype's), an integer zero up to half a step; the result is rounded to the dtype
    u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tol = step * ((0.5 if symmetric else 1.0) + 32 * u) + u * w.double().abs()
    assert ((back - w.double()).abs() <= tol).all()
    assert (back[2] == 0).all()


def test_quantised_layout():
    w = torch.arange(32).float()[None] - 16                     # one row, k = 32
    q, s, z = V.quantize_int4(w, 32)
    assert float(s) == pytest.approx(16 / 7)
    low, high = int(q[0, 0] & 15), int(q[0, 0] >> 4)            # k = 0 low, k = 1 high
    assert low == 8 + round(-16 * 7 / 16) and high == 8 + round(-15 * 7 / 16)


def test_module_keeps_its_state_and_refuses_bad_sizes():
    m = V.Int4Linear.from_weight(torch.randn(10, 64), torch.randn(10), 32, symmetric=False)
    n = V.Int4Linear(64, 10, True, 32, False, torch.float32)
    n.load_state_dict(m.state_dict())
    assert torch.equal(n.dequantized(), m.dequantized()) and torch.equal(n.bias, m.bias)
    with pytest.raises(ValueError, match="multiple of 32"):
        V.Int4Linear(40, 10)
    with pytest.raises(ValueError, match="group_size"):
        V.Int4Linear(64, 10, group_size=48)
    with pytest.raises(ValueError, match="group_size"):
        V.quantize_int4(torch.zeros(2, 64), 16)
    with pytest.raises(AssertionError, match="multiple of 32"):
        V.quantize_int4(torch.zeros(2, 40))


def test_python_api_requires_cuda_tensors():
    x = torch.zeros(1, 32)
    with pytest.raises(AssertionError, match="CUDA"):
        V.int4_linear(x, torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 4), group_size=32)
    with pytest.raises(AssertionError, match="CUDA"):
        V.process_logits(x)
    with pytest.raises(AssertionError, match="CUDA"):
        V.sample_logits(x, temperature=0)


@host_only
def test_int4_linear_rejects_bad_arguments_without_a_device():
    f = _lib.lib().verace_int4_linear
    ok = [FAKE, 64, FAKE, FAKE, None, None, FAKE, 1, 8, 64, 32, 1, 1, None, 0, None]

    def call(**kw):
        names = ["x", "ldx", "q", "s", "z", "bias", "y", "m", "n", "k", "group", "dtype", "out", "ws",
                 "nws", "stream"]
        assert set(kw) <= set(names)
        return f(*[kw.get(n, v) for n, v in zip(names, ok)])

    assert call(group=48) == 2 and "group size 48" in _err()
    assert call(k=40, ldx=40) == 2 and "multiple of 32" in _err()
    assert call(m=-1) == 1 and "negative" in _err()
    assert call(dtype=9, out=9) == 1 and "dtype" in _err()
    assert call(out=2) == 1 and "out_dtype" in _err()
    assert call(ldx=32) == 1 and "row stride" in _err()
    assert call(x=None) == 1 and "NULL" in _err()
    assert call(y=None) == 1 and "NULL" in _err()
    assert call(q=ctypes.c_void_p(264)) == 1 and "aligned" in _err()
    assert call(ldx=68) == 1 and "aligned" in _err()
    size = _lib.lib().verace_int4_linear_workspace
    need = size(64, 4096, 4096, 128, 1)
    assert need > size(64, 4096, 2048, 128, 1) > 0 and size(1, 4096, 1024, 128, 1) == 0 and size(0, 8, 64, 32, 1) == 0
    big = dict(m=64, n=4096, k=4096, ldx=4096, group=128)
    assert call(**big) == 4 and "workspace" in _err()
    assert call(**big, ws=FAKE, nws=need - 1) == 4
    assert call(m=0, x=None, y=None) == 0 and call(n=0, q=None, y=None) == 0       # nothing to do


@host_only
def test_logits_process_rejects_bad_arguments_without_a_device():
    f = _lib.lib().verace_logits_process
    names = ["logits", "ld", "out", "out_ld", "b", "v", "dtype", "odt", "tokens", "tld", "t64", "length", "lengths",
             "prompts", "rp", "r", "pp", "p", "fp", "f", "ids", "values", "n", "i64", "mask", "mld", "stream"]
    ok = [FAKE, 100, ctypes.c_void_p(4096), 100, 2, 100, 0, 0, FAKE, 8, 1, 8, None, None, None, 1.0, None, 0.0, None,
          0.0, None, None, 0, 0, None, 0, None]

    def call(**kw):
        assert set(kw) <= set(names)
        return f(*[kw.get(n, v) for n, v in zip(names, ok)])

    assert call(v=-1) == 1 and "negative" in _err()
    assert call(dtype=5) == 1 and "dtype" in _err()
    assert call(odt=1) == 1 and "out_dtype" in _err()
    assert call(ld=99) == 1 and "row stride" in _err()
    assert call(b=70000) == 2 and "65535" in _err()
    assert call(logits=None) == 1 and "NULL" in _err()
    assert call(tld=7) == 1 and "token row stride" in _err()
    assert call(n=3) == 1 and "bias" in _err()
    assert call(mask=FAKE, mld=3) == 1 and "mask" in _err()
    assert call(out=FAKE, dtype=1, odt=0) == 1 and "in place" in _err()
    assert call(b=0, logits=None, out=None) == 0 and call(v=0, ld=0, out_ld=0) == 0


@host_only
def test_sample_rejects_bad_arguments_without_a_device():
    f = _lib.lib().verace_sample
    names = ["logits", "ld", "noise", "nld", "b", "v", "dtype", "tp", "t", "kp", "k", "pp", "p", "mp", "minp", "tok",
             "lp", "stream"]
    ok = [FAKE, 100, FAKE, 100, 2, 100, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, FAKE, FAKE, None]

    def call(**kw):
        assert set(kw) <= set(names)
        return f(*[kw.get(n, v) for n, v in zip(names, ok)])

    assert call(v=0) == 1 and "empty" in _err()
    assert call(dtype=4) == 1 and "dtype" in _err()
    assert call(noise=None) == 1 and "noise" in _err()
    assert call(noise=None, tp=FAKE, t=0.0) == 1 and "noise" in _err()
    assert call(nld=50) == 1 and "row stride" in _err()
    assert call(tok=None) == 1 and "NULL" in _err()
    assert call(b=0, logits=None) == 0


@host_only
def test_sizes_beyond_32_bit_indices_are_refused_without_a_device():
    """Sizes at which a device index, a stride past the end, would pass 32 bits."""
    L = _lib.lib()
    huge, out = (1 << 30) + 1, ctypes.c_void_p(4096)

    def int4(m, n, k):
        return L.verace_int4_linear(FAKE, k, FAKE, FAKE, None, None, FAKE, m, n, k, 32, 1, 1, None, 0, None)

    assert int4(1, 8, (1 << 31) - 32) == 2 and "too large" in _err()
    assert int4((1 << 20) + 1, 8, 64) == 2 and int4(1, (1 << 28) + 1, 64) == 2
    assert L.verace_int4_linear_workspace(1, 8, (1 << 31) - 32, 32, 1) == 0

    def process(v=100, length=8, biases=0):
        return L.verace_logits_process(FAKE, v, out, v, 2, v, 0, 0, FAKE, length, 1, length, None, None, None, 1.0, None,
                                       0.0, None, 0.0, FAKE, FAKE, biases, 0, None, 0, None)

    for kw in ({"v": huge}, {"length": huge}, {"biases": huge}):
        assert process(**kw) == 2 and "2^30" in _err()
    assert L.verace_sample(FAKE, huge, FAKE, huge, 2, huge, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, FAKE, FAKE,
                           None) == 2 and "2^30" in _err()


def test_package_imports_on_a_torch_without_cuda(monkeypatch):
    """Such a torch lacks the two names that the launch path takes a shortcut through."""
    import importlib
    from verace_v1_b200 import _launch
    for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
        monkeypatch.delattr(torch._C, name, raising=False)
    try:
        again = importlib.reload(_launch)
        assert again.current is torch.cuda.current_device and callable(again.raw_stream)
    finally:
        monkeypatch.undo()
        importlib.reload(_launch)
