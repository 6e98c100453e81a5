"""Dense products of the feed-forward sub-layer with their epilogues in one kernel
(``verace_linear``, ``verace_gated_linear``), forward and backward, and the RMS norm whose
output is in 8 bits (``verace_rmsnorm_fp8``), which feeds them.

The reference runs these as separate steps: ``torch.nn.Linear`` products, the SiTU-GLU
activation (verace_v1/modules/activations.py:8-31), the down projection and the residual's
addition (verace_v1/modules/mcmoe.py:85-120, backbone.py:96-99).

* ``fused_linear``:  act(x Wᵀ + bias) + residual
* ``gated_linear``:  act(x Wgᵀ) up(x Wuᵀ); "situ": beta1 tanh(g / beta1) sigmoid(g) beta2 tanh(u / beta2)
* ``rmsnorm_fp8``, ``add_rmsnorm_fp8``, ``quantize_fp8``: rows as e4m3 values and one fp32 scale each

fp32, bf16 and fp16 operands have gradients; e4m3 operands (with scales) are for inference.
"""
import contextlib
import functools
import math
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._launch import current, raw_stream, wrote
from ._lib import E4M3, F32, check, lib
from .int4 import _require_no_grad
from .kernels import _DTYPE, _norm_args

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_GATES = {"situ": 5, "silu": 2, "gelu": 3, "gelu_tanh": 4, "relu": 1}
FP8 = torch.float8_e4m3fn
_CODE = {**_DTYPE, FP8: E4M3}
_MOST = 1 << 24      # rows and columns of any operand (the C entry points', whose widths are 32-bit)
_ALIGN = {torch.float32: 1, torch.bfloat16: 8, torch.float16: 8, FP8: 16}   # values in 16 bytes (fp32 rows: any)


def _rows(t: torch.Tensor, m: int, k: int) -> Tuple[torch.Tensor, int]:
    """t as [m, k] whose rows the kernels can address, and its row stride; copied where it has to be.  (Rows
    that are not whole 16-byte words may start anywhere.)"""
    a = _ALIGN[t.dtype]
    if t.is_contiguous() and (k % a or a == 1 or t.data_ptr() % 16 == 0):
        return t, k
    if t.dim() != 2:
        t = t.reshape(m, k)
    ld = t.stride(0) if m > 1 else k
    if (k > 1 and t.stride(1) != 1) or ld < k or (k % a == 0 and (ld % a or (a > 1 and t.data_ptr() % 16))):
        if a == 16:     # (copied as bytes)
            t = t.view(torch.uint8).clone(memory_format=torch.contiguous_format).view(FP8)
        else:
            t = t.clone(memory_format=torch.contiguous_format)
        ld = k
    return t, ld


def _vector(t: Optional[torch.Tensor], n: int, dtype: torch.dtype, device, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    assert t.dtype is dtype and t.numel() == n and t.device == device, f"{what} must hold {n} values of {dtype} on {device}"
    return t if t.is_contiguous() else t.contiguous()


def _checked(who, x, weight, scales, want, activation, allowed, out_dtype, default):
    """Checks what both products take (``scales`` of ``want`` are given); returns (activation, k, n, out dtype)."""
    dt = x.dtype
    act = allowed.get(activation)
    assert weight.dim() == 2, f"{who}: the weights must have two dimensions"
    shape, (n, k) = x.shape, weight.shape
    if dt not in _CODE:
        raise ValueError(f"{who}: {dt} inputs (expected fp32, bf16, fp16 or float8_e4m3fn)")
    if act is None:
        raise ValueError(f"{who}: activation {activation!r} (expected one of {tuple(allowed)})")
    assert len(shape) >= 1, "x must have at least one dimension"
    assert weight.dtype is dt and shape[-1] == k and weight.device == x.device, \
        f"{who}: the weights must be [n, {shape[-1]}] in x's dtype, on its device"
    if n > _MOST or k > _MOST:
        raise ValueError(f"{who}: weights of {n} x {k} (at most {_MOST} rows and columns)")
    if dt is FP8:
        if scales != want:
            raise ValueError(f"{who}: float8_e4m3fn operands need their scales, one for x and one for each weight")
        out_dtype = default if out_dtype is None else out_dtype
        if out_dtype not in _DTYPE:
            raise ValueError(f"{who}: out_dtype {out_dtype} for {dt} inputs")
        return act, k, n, out_dtype
    if scales:
        raise ValueError(f"{who}: scales go with float8_e4m3fn operands")
    if out_dtype is None:
        out_dtype = dt
    elif out_dtype is not dt and out_dtype is not torch.float32:
        raise ValueError(f"{who}: out_dtype {out_dtype} for {dt} inputs")
    return act, k, n, out_dtype


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(query: str, m: int, n: int, k: int, code: int) -> int:
    """What the workspace query says, which depends on the sizes and the type alone."""
    return getattr(lib(), query)(m, n, k, code)


def _workspace(nbytes: int, device):
    return torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=device) if nbytes else None


def _no_tangents(who, *tensors):
    """Refuses dual numbers, whose tangents a kernel would drop (called inside of a dual level alone)."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{who} has no forward-mode derivative")


def _output(shape, m, n, dtype, device):
    """Rows of n values in the leading dimensions of x's shape.  (Made in that shape: a view made inside of an autograd
    function may not be changed in place.)"""
    if len(shape) == 2:
        return torch.empty_strided((m, n), (n, 1), dtype=dtype, device=device)
    return torch.empty(shape[:-1] + (n,), dtype=dtype, device=device)


_NOTHING = contextlib.nullcontext()


def _on(dev):
    """The device as the current one (a context; nothing to do where it is)."""
    return _NOTHING if dev.index == current() else torch.cuda.device(dev)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------- act(x Wᵀ + bias) + residual
def _linear(shape, x2, ldx, sx, w2, ldw, sw, bias, res, ldr, m, n, k, act, out_dtype, want_pre):
    dev = x2.device
    y = _output(shape, m, n, out_dtype, dev)
    pre = torch.empty_strided((m, n), (n, 1), dtype=torch.float32, device=dev) if want_pre else None
    L = lib()
    code = _CODE[x2.dtype]
    nws = _workspace_bytes("verace_linear_workspace", m, n, k, code)
    ws = _workspace(nws, dev)
    rc = L.verace_linear(x2.data_ptr(), ldx, _p(sx), w2.data_ptr(), ldw, _p(sw), _p(bias), _p(res), ldr, y.data_ptr(),
                         _p(pre), m, n, k, act, code, _DTYPE[out_dtype], _p(ws), nws, raw_stream(dev.index))
    if rc:
        check(rc, "verace_linear")
    return y, pre


def _fused_linear_backward(ctx, d):
    x2, w2, pre = ctx.saved_tensors
    shape, m, n, k, act, out_dtype = ctx.sizes
    want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
    dx = dw = db = None
    if want_x or want_w or want_b:
        # (what was saved may come back in another layout: hooks move it to the host and back, for one)
        (x2, ldx), (w2, ldw) = _rows(x2, m, k), _rows(w2, n, k)
        if pre is not None:
            pre = pre.contiguous()
        dev, dt = x2.device, x2.dtype
        if want_x:
            dx = _output(shape, m, k, dt, dev)
        if want_w:
            dw = torch.empty_strided((n, k), (k, 1), dtype=dt, device=dev)
        if want_b:
            db = torch.empty_strided((n,), (1,), dtype=dt, device=dev)
        d2 = d.contiguous()
        L = lib()
        code = _DTYPE[dt]
        nws = _workspace_bytes("verace_linear_backward_workspace", m, n, k, code)
        ws = _workspace(nws, dev)
        with _on(dev):
            rc = L.verace_linear_backward(d2.data_ptr(), x2.data_ptr(), ldx, w2.data_ptr(), ldw, _p(pre), _p(dx), _p(dw),
                                          _p(db), m, n, k, act, code, _DTYPE[out_dtype], _p(ws), nws, raw_stream(dev.index))
            if rc:
                check(rc, "verace_linear_backward")
    return dx, dw, db, d if want_r else None, None, None, None, None, None


_fused_linear_backward_once = once_differentiable(_fused_linear_backward)


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype, m, n, k):
        x2, ldx = _rows(x, m, k)
        w2, ldw = _rows(weight, n, k)
        b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        res, ldr = _residual_rows(residual, m, n)
        y, pre = _linear(x.shape, x2, ldx, None, w2, ldw, None, b, res, ldr, m, n, k, act, out_dtype, act != 0)
        ctx.save_for_backward(x2, w2, pre)
        ctx.sizes = (x.shape, m, n, k, act, out_dtype)
        return y

    @staticmethod
    def backward(ctx, d):
        # (where no graph is asked for, without the wrapper that refuses the second derivative: 6 us)
        return (_fused_linear_backward_once if torch.is_grad_enabled() else _fused_linear_backward)(ctx, d)


def _residual_rows(residual, m, n):
    if residual is None:
        return None, n
    r = residual if residual.dim() == 2 else residual.reshape(m, n)
    if (n > 1 and r.stride(1) != 1) or (m > 1 and r.stride(0) < n):
        r = r.contiguous()
    return r, r.stride(0) if m > 1 else n


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                 x_scale: Optional[torch.Tensor] = None, w_scale: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x weightᵀ + bias) + residual in one kernel: x [..., k], weight [n, k], bias [n] (x's dtype),
    residual [..., n] (the output's dtype); activation None, "relu", "silu", "gelu" (by erf) or "gelu_tanh".
    The output has x's dtype or, with ``out_dtype=torch.float32``, fp32; sums are fp32, rounded once.  fp32 operands keep
    their 24 bits; an infinity in them gives NaN (that of the formula with up to 24 rows of x).

    With float8_e4m3fn x and weight, ``x_scale`` (one fp32 value a row of x) and ``w_scale`` [n] multiply
    them; the output is then fp32, bf16 or fp16 (``out_dtype``, else the residual's dtype, else bf16), the bias of
    the same dtype.  The other types are differentiable in x, weight, bias and residual (once)."""
    dev = x.device
    if dev.index is None or dev.index != current():
        assert x.is_cuda, "This kernel requires CUDA tensors"
        with torch.cuda.device(dev):
            return fused_linear(x, weight, bias, activation=activation, residual=residual, x_scale=x_scale,
                                w_scale=w_scale, out_dtype=out_dtype)
    act, k, n, odt = _checked("fused_linear", x, weight, (x_scale is not None) + (w_scale is not None), 2, activation,
                              _ACTIVATIONS, out_dtype, torch.bfloat16 if residual is None else residual.dtype)
    lead = x.shape[:-1]
    m = lead[0] if len(lead) == 1 else math.prod(lead)
    eight = x.dtype is FP8
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
    b = bias
    if bias is not None:
        bias_dtype = odt if eight else x.dtype
        assert bias.dtype is bias_dtype and bias.shape == (n,) and bias.device == dev, \
            f"bias must be [{n}] in {bias_dtype}, on x's device"
        grad = grad or bias.requires_grad and torch.is_grad_enabled()
        if not bias.is_contiguous():
            b = bias.contiguous()
    if residual is not None:
        assert residual.shape == lead + (n,) and residual.dtype is odt and residual.device == dev, \
            f"residual must be {tuple(lead) + (n,)} in {odt}, on x's device"
        grad = grad or residual.requires_grad and torch.is_grad_enabled()
    if forward_ad._current_level >= 0:
        _no_tangents("fused_linear", x, weight, bias, residual, x_scale, w_scale)
    if eight and (x_scale.requires_grad or w_scale.requires_grad):
        grad = torch.is_grad_enabled()
    if grad:
        if eight:
            raise RuntimeError("fused_linear runs 8-bit operands for inference (no autograd path): "
                               "call it under torch.no_grad()")
        return _FusedLinear.apply(x, weight, bias, residual, act, odt, m, n, k)
    x2, ldx = _rows(x, m, k)
    w2, ldw = _rows(weight, n, k)
    sx = sw = None
    if eight:
        sx = _vector(x_scale, m, torch.float32, dev, "x_scale")
        sw = _vector(w_scale, n, torch.float32, dev, "w_scale")
    res, ldr = _residual_rows(residual, m, n)
    return _linear(x.shape, x2, ldx, sx, w2, ldw, sw, b, res, ldr, m, n, k, act, odt, False)[0]


# ---------------------------------------------------------------------------- act(x Wgᵀ) up(x Wuᵀ)
def _gate_rows(w_gate, w_up, f, k):
    g2, ldg = _rows(w_gate, f, k)
    u2, ldu = _rows(w_up, f, k)
    if ldg != ldu:      # (two row strides: the one that is not dense, or both, become so)
        if ldg != k:
            g2, ldg = _rows(w_gate.contiguous(), f, k)
        if ldu != k:
            u2, ldu = _rows(w_up.contiguous(), f, k)
    return g2, u2, ldg


def _gated(shape, x2, ldx, sx, g2, u2, ldw, sg, su, m, f, k, act, b1, b2, out_dtype, want_pre):
    dev = x2.device
    h = _output(shape, m, f, out_dtype, dev)
    gate = up = None
    if want_pre:
        gate = torch.empty_strided((m, f), (f, 1), dtype=torch.float32, device=dev)
        up = torch.empty_strided((m, f), (f, 1), dtype=torch.float32, device=dev)
    L = lib()
    code = _CODE[x2.dtype]
    nws = _workspace_bytes("verace_gated_linear_workspace", m, f, k, code)
    ws = _workspace(nws, dev)
    rc = L.verace_gated_linear(x2.data_ptr(), ldx, _p(sx), g2.data_ptr(), u2.data_ptr(), ldw, _p(sg), _p(su), h.data_ptr(),
                               _p(gate), _p(up), m, f, k, act, b1, b2, code, _DTYPE[out_dtype], _p(ws), nws,
                               raw_stream(dev.index))
    if rc:
        check(rc, "verace_gated_linear")
    return h, gate, up


def _gated_linear_backward(ctx, d):
    x2, g2, u2, gate, up = ctx.saved_tensors
    shape, m, f, k, act, b1, b2, out_dtype = ctx.sizes
    want_x, want_g, want_u = ctx.needs_input_grad[:3]
    (x2, ldx), (g2, u2, ldw) = _rows(x2, m, k), _gate_rows(g2, u2, f, k)     # (as in _fused_linear_backward)
    gate, up = gate.contiguous(), up.contiguous()
    dev, dt = x2.device, x2.dtype
    dx = _output(shape, m, k, dt, dev) if want_x else None
    dg = torch.empty_strided((f, k), (k, 1), dtype=dt, device=dev) if want_g else None
    du = torch.empty_strided((f, k), (k, 1), dtype=dt, device=dev) if want_u else None
    d2 = d.contiguous()
    L = lib()
    code = _DTYPE[dt]
    nws = _workspace_bytes("verace_gated_linear_backward_workspace", m, f, k, code)
    ws = _workspace(nws, dev)
    with _on(dev):
        rc = L.verace_gated_linear_backward(d2.data_ptr(), x2.data_ptr(), ldx, g2.data_ptr(), u2.data_ptr(), ldw,
                                            gate.data_ptr(), up.data_ptr(), _p(dx), _p(dg), _p(du), m, f, k, act, b1, b2, code,
                                            _DTYPE[out_dtype], _p(ws), nws, raw_stream(dev.index))
        if rc:
            check(rc, "verace_gated_linear_backward")
    return dx, dg, du, None, None, None, None, None, None, None


_gated_linear_backward_once = once_differentiable(_gated_linear_backward)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act, b1, b2, out_dtype, m, f, k):
        x2, ldx = _rows(x, m, k)
        g2, u2, ldw = _gate_rows(w_gate, w_up, f, k)
        h, gate, up = _gated(x.shape, x2, ldx, None, g2, u2, ldw, None, None, m, f, k, act, b1, b2, out_dtype, True)
        ctx.save_for_backward(x2, g2, u2, gate, up)
        ctx.sizes = (x.shape, m, f, k, act, b1, b2, out_dtype)
        return h

    @staticmethod
    def backward(ctx, d):
        return (_gated_linear_backward_once if torch.is_grad_enabled() else _gated_linear_backward)(ctx, d)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = "situ",
                 beta1: float = 4.0, beta2: float = 25.0, x_scale: Optional[torch.Tensor] = None,
                 gate_scale: Optional[torch.Tensor] = None, up_scale: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(g) up(u) with g = x w_gateᵀ and u = x w_upᵀ in one kernel: x [..., k], w_gate and w_up [f, k] ->
    [..., f].  activation "situ" (``SiTUGLU``: beta1 tanh(g / beta1) sigmoid(g) beta2 tanh(u / beta2)), or "silu",
    "gelu" (by erf), "gelu_tanh" or "relu" of g, times u.  g and u stay in fp32; the result is rounded once, to
    x's dtype or, with ``out_dtype=torch.float32``, not at all.

    With float8_e4m3fn operands, ``x_scale`` (one fp32 value a row of x), ``gate_scale`` and ``up_scale`` [f]
    multiply them, and the output is fp32, bf16 (the default) or fp16.  The other types are differentiable in x, w_gate
    and w_up (once); the pass keeps g and u, in fp32, for the backward."""
    dev = x.device
    if dev.index is None or dev.index != current():
        assert x.is_cuda, "This kernel requires CUDA tensors"
        with torch.cuda.device(dev):
            return gated_linear(x, w_gate, w_up, activation=activation, beta1=beta1, beta2=beta2, x_scale=x_scale,
                                gate_scale=gate_scale, up_scale=up_scale, out_dtype=out_dtype)
    act, k, f, odt = _checked("gated_linear", x, w_gate, (x_scale is not None) + (gate_scale is not None)
                              + (up_scale is not None), 3, activation, _GATES, out_dtype, torch.bfloat16)
    assert w_up.shape == w_gate.shape and w_up.dtype is w_gate.dtype and w_up.device == dev, \
        "gated_linear: the weights must be two of one shape and dtype, on x's device"
    if act == 5 and not (beta1 and beta2):
        raise ValueError(f"gated_linear: beta1 {beta1}, beta2 {beta2} (expected anything but 0)")
    lead = x.shape[:-1]
    m = lead[0] if len(lead) == 1 else math.prod(lead)
    eight = x.dtype is FP8
    if forward_ad._current_level >= 0:
        _no_tangents("gated_linear", x, w_gate, w_up, x_scale, gate_scale, up_scale)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or eight and (x_scale.requires_grad or gate_scale.requires_grad or up_scale.requires_grad)):
        if eight:
            raise RuntimeError("gated_linear runs 8-bit operands for inference (no autograd path): "
                               "call it under torch.no_grad()")
        return _GatedLinear.apply(x, w_gate, w_up, act, float(beta1), float(beta2), odt, m, f, k)
    x2, ldx = _rows(x, m, k)
    g2, u2, ldw = _gate_rows(w_gate, w_up, f, k)
    sx = sg = su = None
    if eight:
        sx = _vector(x_scale, m, torch.float32, dev, "x_scale")
        sg = _vector(gate_scale, f, torch.float32, dev, "gate_scale")
        su = _vector(up_scale, f, torch.float32, dev, "up_scale")
    return _gated(x.shape, x2, ldx, sx, g2, u2, ldw, sg, su, m, f, k, act, beta1, beta2, odt, False)[0]


# ---------------------------------------------------------------------------- rows in 8 bits
def _to_fp8(who, h, y, sum_out, norm, return_norm):
    """The rows of h (of h + y, which goes to sum_out) in 8 bits; norm None: as they are.  All contiguous."""
    dt, shape = h.dtype, h.shape
    code = _DTYPE.get(dt)
    if code is None:
        raise ValueError(f"{who}: {dt} inputs (expected fp32, bf16 or fp16)")
    assert len(shape) >= 1 and shape[-1] > 0, f"{who}: rows of at least one value"
    if shape[-1] > _MOST:
        raise ValueError(f"{who}: rows of {shape[-1]} columns (at most 32768)")
    if h.requires_grad:
        _require_no_grad(h, who)
    if forward_ad._current_level >= 0:
        _no_tangents(who, h, y, None if norm is None else norm.weight)
    dev, cols = h.device, shape[-1]
    w, eps = (None, 0.0) if norm is None else _norm_args(norm, h)
    q = torch.empty_like(h, dtype=FP8)
    if len(shape) == 2:
        scale = torch.empty_strided(shape[:1], (1,), dtype=torch.float32, device=dev)
    else:
        scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    n = torch.empty_like(h) if return_norm else None
    rc = lib().verace_rmsnorm_fp8(h.data_ptr(), None if y is None else y.data_ptr(),
                                  None if y is None else sum_out.data_ptr(), w or None, eps, 0 if norm is None else 1,
                                  q.data_ptr(), scale.data_ptr(), None if n is None else n.data_ptr(), h.numel() // cols,
                                  cols, code, raw_stream(dev.index))
    if rc:
        check(rc, who)
    return (q, scale, n) if return_norm else (q, scale)


def quantize_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows of x [..., k] (fp32, bf16 or fp16; k up to 32761, or 32768) as (float8_e4m3fn [..., k], fp32 scales [...]):
    scale = max(max |x|, 2^-100) / 448 of the row, values rounded to the nearest."""
    dev = x.device
    if dev.index is None or dev.index != current():
        assert x.is_cuda, "This kernel requires CUDA tensors"
        with torch.cuda.device(x.device):
            return quantize_fp8(x)
    return _to_fp8("quantize_fp8", x.contiguous(), None, None, None, False)


def rmsnorm_fp8(x: torch.Tensor, norm: nn.RMSNorm, *, return_norm: bool = False):
    """``norm`` (a torch.nn.RMSNorm over the last dimension) applied to x, its rows in 8 bits as
    ``quantize_fp8`` gives them: (q, scale), and with ``return_norm`` the norm's output in x's dtype as well.
    The values are not rounded to x's dtype before they are rounded to 8 bits."""
    dev = x.device
    if dev.index is None or dev.index != current():
        assert x.is_cuda, "This kernel requires CUDA tensors"
        with torch.cuda.device(x.device):
            return rmsnorm_fp8(x, norm, return_norm=return_norm)
    return _to_fp8("rmsnorm_fp8", x.contiguous(), None, None, norm, return_norm)


def add_rmsnorm_fp8(h: torch.Tensor, y: torch.Tensor, norm: nn.RMSNorm, *, out: Optional[torch.Tensor] = None,
                    return_norm: bool = False):
    """A block's residual step ahead of 8-bit products, in one pass: h <- h + y in place (or into ``out``),
    then ``rmsnorm_fp8`` of the sum: (q, scale), and with ``return_norm`` the norm's output as well."""
    dev = h.device
    if dev.index is None or dev.index != current():
        assert h.is_cuda, "This kernel requires CUDA tensors"
        with torch.cuda.device(dev):
            return add_rmsnorm_fp8(h, y, norm, out=out, return_norm=return_norm)
    if y.requires_grad:
        _require_no_grad(y, "add_rmsnorm_fp8")
    assert y.shape == h.shape and y.dtype is h.dtype and y.device == dev, "h and y must match"
    if out is None:
        out = h
    elif out is not h:
        assert out.shape == h.shape and out.dtype is h.dtype and out.device == dev, \
            "the sum goes to a tensor of h's shape, dtype and device"
        if out.requires_grad:
            _require_no_grad(out, "add_rmsnorm_fp8")
    assert out.is_contiguous(), "the sum goes to a contiguous tensor"
    made = _to_fp8("add_rmsnorm_fp8", h.contiguous(), y.contiguous(), out, norm, return_norm)
    wrote(out)
    return made


# ---------------------------------------------------------------------------- modules with 8-bit weights
Rows8 = Tuple[torch.Tensor, torch.Tensor]     # e4m3 rows and their scales


def _rows8(x) -> Rows8:
    return x if isinstance(x, tuple) else quantize_fp8(x)


class _Fp8Module(nn.Module):
    """A module with e4m3 weights.  ``to``, ``half`` and the like change the type of its outputs (``dtype``) and bias; the
    8-bit values and their fp32 scales keep theirs and move between devices with it (torch counts 8-bit values as
    floating point and would cast them)."""
    _packed: Tuple[str, ...] = ()

    def _apply(self, fn, recurse: bool = True):
        held = {name: self._buffers[name] for name in self._packed}
        device = held[self._packed[0]].device
        self._buffers.update(dict.fromkeys(held))
        try:
            super()._apply(fn, recurse)
            for name, t in held.items():
                bits = fn(t.view(torch.uint8 if t.dtype is FP8 else torch.int32))
                held[name] = bits.view(t.dtype) if not bits.is_floating_point() else t.to(bits.device)
            self.dtype = fn(torch.empty(0, dtype=self.dtype, device=device)).dtype
        finally:
            self._buffers.update(held)
        return self


class Fp8Linear(_Fp8Module):
    """A linear layer with e4m3 weights (buffers ``weight``, ``scales``, ``bias``) in place of a
    ``torch.nn.Linear``.  Its input is a tensor, whose rows it quantises, or rows in 8 bits as
    ``rmsnorm_fp8`` gives them: (values, scales).  The output has ``dtype``."""
    _packed = ("weight", "scales")

    def __init__(self, in_features: int, out_features: int, bias: bool = False, dtype: torch.dtype = torch.bfloat16,
                 device=None):
        super().__init__()
        self.in_features, self.out_features, self.dtype = in_features, out_features, dtype
        self.register_buffer("weight", torch.zeros(out_features, in_features, dtype=FP8, device=device))
        self.register_buffer("scales", torch.zeros(out_features, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Fp8Linear":
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, linear.weight.dtype, device="meta")
        m.weight, m.scales = quantize_fp8(linear.weight.detach())
        m.bias = None if linear.bias is None else linear.bias.detach().clone()
        return m

    def forward(self, x, residual: Optional[torch.Tensor] = None, activation: Optional[str] = None) -> torch.Tensor:
        q, s = _rows8(x)
        return fused_linear(q, self.weight, self.bias, activation=activation, residual=residual, x_scale=s,
                            w_scale=self.scales, out_dtype=self.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class Fp8GatedLinear(_Fp8Module):
    """The gate and up projections of a gated block with e4m3 weights and the gate in their product's epilogue
    (buffers ``w_gate``, ``w_up``, ``gate_scales``, ``up_scales``); its input is as ``Fp8Linear``'s."""
    _packed = ("w_gate", "w_up", "gate_scales", "up_scales")

    def __init__(self, in_features: int, hidden_features: int, activation: str = "situ", beta1: float = 4.0,
                 beta2: float = 25.0, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        self.in_features, self.hidden_features, self.dtype = in_features, hidden_features, dtype
        self.activation, self.beta1, self.beta2 = activation, beta1, beta2
        for w, s in (("w_gate", "gate_scales"), ("w_up", "up_scales")):
            self.register_buffer(w, torch.zeros(hidden_features, in_features, dtype=FP8, device=device))
            self.register_buffer(s, torch.zeros(hidden_features, device=device))

    @classmethod
    def from_weights(cls, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "situ", beta1: float = 4.0,
                     beta2: float = 25.0) -> "Fp8GatedLinear":
        f, k = w_gate.shape
        m = cls(k, f, activation, beta1, beta2, w_gate.dtype, device="meta")
        m.w_gate, m.gate_scales = quantize_fp8(w_gate.detach())
        m.w_up, m.up_scales = quantize_fp8(w_up.detach())
        return m

    def forward(self, x) -> torch.Tensor:
        q, s = _rows8(x)
        return gated_linear(q, self.w_gate, self.w_up, activation=self.activation, beta1=self.beta1, beta2=self.beta2,
                            x_scale=s, gate_scale=self.gate_scales, up_scale=self.up_scales, out_dtype=self.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, hidden_features={self.hidden_features}, activation={self.activation}"


def _check_weights(*weights: torch.Tensor):
    """Refuses weights that ``quantize_fp8`` does not take."""
    for w in weights:
        assert w.is_cuda, "This kernel requires CUDA tensors"
        if w.dtype not in _DTYPE:
            raise ValueError(f"quantize_model_fp8: {w.dtype} weights (expected fp32, bf16 or fp16)")
        if w.shape[1] > 32761 and w.shape[1] != 32768:
            raise ValueError(f"quantize_model_fp8: weights of {w.shape[1]} inputs (at most 32761, or 32768)")


def quantize_model_fp8(model: nn.Module, lm_head: bool = True) -> nn.Module:
    """Puts the feed-forward sub-layers of a model (a ``VeraceV1Model``, ``VeraceV1Layer`` or any module that
    holds the framework's M-CMoE) into 8 bits, in place, and with ``lm_head`` the LM head (the token embedding
    keeps its own table): the gate and up projections with the gate in their epilogue, the down projection with the
    manifold's part in its epilogue; inside a layer the norm before the sub-layer writes the rows in 8 bits along
    with the residual's addition.  The model must be on a CUDA device; the dense weights are dropped.  Routers, the
    sigma projection, norms, bases and the mixers stay as they are, and so does what ``quantize_model_int4`` has
    put into 4 bits.  A model that cannot go into 8 bits as a whole is refused as it is."""
    from .mcmoe import ManifoldContinuousMoE, SiTUGLU

    modules = list(model.modules())
    lm_head = lm_head and isinstance(getattr(model, "lm_head", None), nn.Linear)
    for m in modules:
        if isinstance(m, SiTUGLU) and m.fp8_in is None and m.int4_in is None:
            _check_weights(m.w_gate.weight, m.w_up.weight)
        elif isinstance(m, ManifoldContinuousMoE) and isinstance(m.base_w_down, nn.Linear):
            _check_weights(m.base_w_down.weight)
    if lm_head:
        _check_weights(model.lm_head.weight)
    for m in modules:
        if isinstance(m, SiTUGLU) and m.fp8_in is None and m.int4_in is None:
            m.fp8_in = Fp8GatedLinear.from_weights(m.w_gate.weight, m.w_up.weight, "situ", m.beta1, m.beta2)
            m.w_gate = m.w_up = None
            m._stacked = m._stacked_key = None
        elif isinstance(m, ManifoldContinuousMoE) and isinstance(m.base_w_down, nn.Linear):
            m.base_w_down = Fp8Linear.from_linear(m.base_w_down)
    if lm_head:
        model.lm_head = Fp8Linear.from_linear(model.lm_head)
    return model
