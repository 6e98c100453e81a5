"""CPU checks of the dense products with epilogues and the 8-bit norm: what the entry points refuse
(placeholder pointers only where no GPU is visible)."""
import ctypes

import pytest
import torch

import verace_v1_b200 as V
from verace_v1_b200 import _lib

host_only = pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers: run without a GPU only")
FAKE, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)


def _err():
    return _lib.lib().verace_last_error().decode()


def caller(name, names, ok):
    f = getattr(_lib.lib(), name)

    def call(**kw):
        args = dict(zip(names, ok))
        assert set(kw) <= set(args)
        args.update(kw)
        return f(*args.values())
    return call


def test_python_api_requires_cuda_tensors():
    x, w = torch.zeros(2, 16), torch.zeros(4, 16)
    norm = torch.nn.RMSNorm(16)
    for call in (lambda: V.fused_linear(x, w), lambda: V.gated_linear(x, w, w), lambda: V.quantize_fp8(x),
                 lambda: V.rmsnorm_fp8(x, norm), lambda: V.add_rmsnorm_fp8(x, x, norm)):
        with pytest.raises(AssertionError, match="CUDA"):
            call()


@host_only
def test_norm_rejects_bad_arguments_without_a_device():
    call = caller("verace_rmsnorm_fp8", ["h", "y", "sum", "w", "eps", "norm", "q", "scale", "n", "rows", "cols", "dtype",
                                         "stream"], [FAKE, FAKE, FAKE, FAKE, 1e-6, 1, FAKE, FAKE, None, 2, 64, 1, None])
    for kw, rc, text in [({"rows": -1}, 1, "rows"), ({"cols": 0}, 1, "cols"), ({"dtype": 3}, 1, "dtype"),
                         ({"cols": 32769}, 2, "32768"), ({"h": None}, 1, "NULL"), ({"q": None}, 1, "NULL"),
                         ({"sum": None}, 1, "sum"), ({"y": None}, 1, "sum")]:
        assert call(**kw) == rc and text in _err(), kw
    assert call(rows=0) == 0


@host_only
def test_linear_rejects_bad_arguments_without_a_device():
    names = ["x", "ldx", "sx", "w", "ldw", "sw", "bias", "res", "ldr", "out", "pre", "m", "n", "k", "act", "dtype", "odt",
             "ws", "nws", "stream"]
    call = caller("verace_linear", names, [FAKE, 64, None, FAKE, 64, None, None, None, 8, FAKE, None, 4, 8, 64, 0, 1, 1,
                                           None, 0, None])
    for kw, rc, text in [({"m": -1}, 1, "negative"), ({"k": 1 << 25}, 2, "too large"), ({"act": 5}, 1, "activation"),
                         ({"dtype": 4}, 1, "dtype"), ({"odt": 2}, 1, "out_dtype"), ({"x": None}, 1, "NULL x"),
                         ({"ldx": 32}, 1, "row stride"), ({"ldw": 68}, 1, "aligned"), ({"w": ODD}, 1, "aligned"),
                         ({"out": None}, 1, "NULL out"), ({"sx": FAKE}, 1, "scales"), ({"dtype": 3}, 1, "scales"),
                         ({"res": FAKE, "ldr": 4}, 1, "residual")]:
        assert call(**kw) == rc and text in _err(), kw
    assert call(m=0) == 0 and call(n=0) == 0
    back = caller("verace_linear_backward", ["d", "x", "ldx", "w", "ldw", "pre", "dx", "dw", "db", "m", "n", "k", "act", "dtype",
                                             "odt", "ws", "nws", "stream"],
                  [FAKE, FAKE, 64, FAKE, 64, FAKE, FAKE, FAKE, FAKE, 4, 8, 64, 2, 1, 1, FAKE, 1 << 20, None])
    for kw, rc, text in [({"d": None}, 1, "NULL"), ({"pre": None}, 1, "NULL"), ({"dtype": 3, "odt": 1}, 1, "dtype"),
                         ({"x": ODD}, 1, "aligned"), ({"ws": None}, 4, "workspace"), ({"nws": 16}, 4, "workspace")]:
        assert back(**kw) == rc and text in _err(), kw


@host_only
def test_gated_linear_rejects_bad_arguments_without_a_device():
    names = ["x", "ldx", "sx", "wg", "wu", "ldw", "sg", "su", "out", "gate", "up", "m", "f", "k", "act", "b1", "b2", "dtype",
             "odt", "ws", "nws", "stream"]
    call = caller("verace_gated_linear", names, [FAKE, 64, None, FAKE, FAKE, 64, None, None, FAKE, None, None, 4, 8, 64, 5, 4.0,
                                                 25.0, 1, 1, None, 0, None])
    for kw, rc, text in [({"f": -1}, 1, "negative"), ({"act": 0}, 1, "activation"), ({"act": 6}, 1, "activation"),
                         ({"b2": 0.0}, 1, "beta"), ({"wu": None}, 1, "w_up"), ({"wg": ODD}, 1, "aligned"),
                         ({"gate": FAKE}, 1, "one of gate and up"), ({"dtype": 3}, 1, "scales"),
                         ({"odt": 3}, 1, "out_dtype")]:
        assert call(**kw) == rc and text in _err(), kw
    back = caller("verace_gated_linear_backward", ["d", "x", "ldx", "wg", "wu", "ldw", "gate", "up", "dx", "dg", "du", "m", "f",
                                                   "k", "act", "b1", "b2", "dtype", "odt", "ws", "nws", "stream"],
                  [FAKE, FAKE, 64, FAKE, FAKE, 64, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 64, 5, 4.0, 25.0, 1, 1, FAKE, 1 << 20,
                   None])
    for kw, rc, text in [({"gate": None}, 1, "NULL"), ({"b1": 0.0}, 1, "beta"), ({"dtype": 3, "odt": 1}, 1, "dtype"),
                         ({"nws": 16}, 4, "workspace")]:
        assert back(**kw) == rc and text in _err(), kw


def test_workspaces_grow_with_the_problem():
    L = _lib.lib()
    for name in ("verace_linear_backward_workspace", "verace_gated_linear_backward_workspace"):
        f = getattr(L, name)
        for dtype in (0, 1, 2):
            assert 0 < f(64, 128, 64, dtype) < f(1024, 128, 64, dtype) < f(1024, 4096, 64, dtype)
        assert f(64, 128, 64, 1) < f(64, 128, 64, 0)
