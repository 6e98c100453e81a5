"""Products with 4-bit weights for the decode step (``verace_int4_linear``).

The reference's projections and LM head are dense ``torch.nn.Linear`` products
(verace_v1/modules/backbone.py:202, sssd_attention.py:116-126).  A decode step of a few
sequences reads every weight for a handful of multiplications, so its time is the weights'
bytes; codes of 4 bits with one scale (and zero) per group of 32, 64 or 128 inputs are a
quarter of bf16's.

Layout, as :func:`quantize_int4` makes it: ``qweight`` uint8 [n, k/2], two codes to a byte
along k, the even k in the low half; ``scales`` [ceil(k/group), n] in the activations'
dtype; ``zeros`` uint8 [ceil(k/group), n], 0 to 15, or None (8 everywhere).
W[n, k] = scales[k // group, n] * (code - zero).
"""
from typing import Optional, Tuple

import torch
import torch.nn as nn

from ._lib import F32, check, lib
from .kernels import _DTYPE
from ._launch import current, raw_stream

GROUP_SIZES = (32, 64, 128)
_SIZE = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2}


def _require_no_grad(x: torch.Tensor, who: str):
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{who} runs for inference (no autograd path): call it under torch.no_grad()")


def _check_packed(qweight, scales, zeros, bias, k, group_size, dtype):
    """Checks a packed weight against the inputs' width and dtype; returns its number of rows."""
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size {group_size}: expected one of {GROUP_SIZES}")
    assert k % 32 == 0, "the input width must be a multiple of 32"
    assert qweight.dtype is torch.uint8 and qweight.dim() == 2 and qweight.shape[1] * 2 == k, \
        "qweight must be uint8 [n, k / 2]"
    n = qweight.shape[0]
    shape = (-(-k // group_size), n)
    assert scales.dtype is dtype and scales.shape == shape, \
        "scales must be [ceil(k / group_size), n] in the activations' dtype"
    assert zeros is None or (zeros.dtype is torch.uint8 and zeros.shape == shape), \
        "zeros must be uint8 in the shape of scales"
    assert bias is None or (bias.dtype is dtype and bias.shape == (n,)), "bias must be [n] in the activations' dtype"
    return n


def int4_linear(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,
                zeros: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                group_size: int = 128, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., k] (fp32, bf16 or fp16) times the 4-bit weight's transpose, plus bias: [..., n]
    in x's dtype or, with ``out_dtype=torch.float32``, in fp32.  Sums are fp32, the output is
    rounded once; inputs below 2^-13 of their row's largest may be off by up to 2^-21 of it (bf16;
    2^-23 fp16, 2^-37 fp32).  Any number of rows; meant for the few of a decode step."""
    assert x.is_cuda, "This kernel requires CUDA tensors"
    if x.requires_grad:
        _require_no_grad(x, "int4_linear")
    dev = x.device
    index = dev.index
    if index != current():
        with torch.cuda.device(dev):
            return int4_linear(x, qweight, scales, zeros, bias, group_size=group_size, out_dtype=out_dtype)
    dt = x.dtype
    code = _DTYPE.get(dt)
    if code is None:
        raise ValueError(f"int4_linear: {dt} activations (expected fp32, bf16 or fp16)")
    if out_dtype is None or out_dtype is dt:
        odt, ocode = dt, code
    elif out_dtype is torch.float32:
        odt, ocode = out_dtype, F32
    else:
        raise ValueError(f"int4_linear: out_dtype {out_dtype} (expected {dt} or torch.float32)")
    shape = x.shape
    k = shape[-1]
    n = _check_packed(qweight, scales, zeros, bias, k, group_size, dt)
    flat = len(shape) == 2
    x2 = x if flat else x.reshape(-1, k)
    m, ldx = x2.shape[0], k
    xp = x2.data_ptr()
    if m > 1:
        ldx = x2.stride(0)
    if xp % 16 or (k > 1 and x2.stride(1) != 1) or ldx < k or ldx * _SIZE[dt] % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
        xp, ldx = x2.data_ptr(), k
    qp = qweight.data_ptr()
    if qp % 16 or not qweight.is_contiguous():
        qweight = qweight.clone(memory_format=torch.contiguous_format)
        qp = qweight.data_ptr()
    if not scales.is_contiguous():
        scales = scales.contiguous()
    zp = bp = None
    if zeros is not None:
        if not zeros.is_contiguous():
            zeros = zeros.contiguous()
        zp = zeros.data_ptr()
    if bias is not None:
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bp = bias.data_ptr()
    assert qweight.device == dev and scales.device == dev and (zp is None or zeros.device == dev) \
        and (bp is None or bias.device == dev), "all tensors must be on one device"
    y = x.new_empty((m, n), dtype=odt)
    L = lib()
    nws = L.verace_int4_linear_workspace(m, n, k, group_size, code)
    wp = None
    if nws:
        ws = x.new_empty(nws, dtype=torch.uint8)
        wp = ws.data_ptr()
    rc = L.verace_int4_linear(xp, ldx, qp, scales.data_ptr(), zp, bp, y.data_ptr(), m, n, k, group_size, code, ocode,
                              wp, nws, raw_stream(index))
    if rc:
        check(rc, "verace_int4_linear")
    return y if flat else y.view(shape[:-1] + (n,))


def quantize_int4(weight: torch.Tensor, group_size: int = 128, symmetric: bool = True
                  ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(qweight, scales, zeros) of weight [n, k]: round-to-nearest codes per group of
    ``group_size`` along k.  Symmetric: scale = max |w| / 7, no zeros.  Otherwise the range
    [min(w, 0), max(w, 0)] on 15 steps with an integer zero.  The scales are rounded to the
    weight's dtype before the codes are taken."""
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size {group_size}: expected one of {GROUP_SIZES}")
    assert weight.dim() == 2 and weight.shape[1] % 32 == 0, "weight must be [n, k] with k a multiple of 32"
    n, k = weight.shape
    groups = -(-k // group_size)
    w = weight.detach().float()
    pad = groups * group_size - k
    w = torch.nn.functional.pad(w, (0, pad)).view(n, groups, group_size)
    if symmetric:
        s = w.abs().amax(-1) / 7
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        s = (hi - lo) / 15
    s = s.to(weight.dtype)
    sf = s.float()
    inv = torch.where(sf > 0, 1 / sf, torch.zeros_like(sf))
    z = torch.full_like(sf, 8.0) if symmetric else torch.round(-lo * inv).clamp_(0, 15)
    q = (torch.round(w * inv.unsqueeze(-1)) + z.unsqueeze(-1)).clamp_(0, 15).to(torch.uint8)
    q = q.view(n, -1)[:, :k]
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    return packed.contiguous(), s.t().contiguous(), None if symmetric else z.to(torch.uint8).t().contiguous()


def dequantize_int4(qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
                    group_size: int = 128) -> torch.Tensor:
    """The weight [n, k] that the codes stand for, in the scales' dtype (computed in fp32)."""
    n, k = qweight.shape[0], qweight.shape[1] * 2
    _check_packed(qweight, scales, zeros, None, k, group_size, scales.dtype)
    q = torch.stack((qweight & 15, qweight >> 4), dim=-1).view(n, k).float()
    of = torch.arange(k, device=q.device) // group_size
    z = 8.0 if zeros is None else zeros.float().t()[:, of]
    return ((q - z) * scales.float().t()[:, of]).to(scales.dtype)


class Int4Linear(nn.Module):
    """A linear layer with 4-bit weights (buffers ``qweight``, ``scales``, ``zeros``, ``bias``)
    in place of a ``torch.nn.Linear``."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, group_size: int = 128,
                 symmetric: bool = True, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size {group_size}: expected one of {GROUP_SIZES}")
        if in_features % 32:
            raise ValueError(f"in_features {in_features}: expected a multiple of 32")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        groups = -(-in_features // group_size)
        self.register_buffer("qweight", torch.zeros(out_features, in_features // 2, dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros(groups, out_features, dtype=dtype, device=device))
        self.register_buffer("zeros", None if symmetric else
                             torch.zeros(groups, out_features, dtype=torch.uint8, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, group_size: int = 128,
                    symmetric: bool = True) -> "Int4Linear":
        n, k = weight.shape
        m = cls(k, n, bias is not None, group_size, symmetric, weight.dtype, device="meta")
        m.qweight, m.scales, m.zeros = quantize_int4(weight, group_size, symmetric)
        m.bias = None if bias is None else bias.detach().clone()
        return m

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 128, symmetric: bool = True) -> "Int4Linear":
        return cls.from_weight(linear.weight, linear.bias, group_size, symmetric)

    def dequantized(self) -> torch.Tensor:
        return dequantize_int4(self.qweight, self.scales, self.zeros, group_size=self.group_size)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int4_linear(x, self.qweight, self.scales, self.zeros, self.bias, group_size=self.group_size)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, group_size={self.group_size}, "
                f"zeros={self.zeros is not None}, bias={self.bias is not None}")


def quantize_model_int4(model: nn.Module, group_size: int = 128, symmetric: bool = True,
                        lm_head: bool = True) -> nn.Module:
    """Puts the projections of a model's layers (a ``VeraceV1Model``, ``VeraceV1Layer`` or any module
    that holds the framework's mixers and M-CMoE) into 4 bits, in place: the concatenated input
    projections of both mixers and the stacked gate / up projection as one weight each, the
    output projections, the M-CMoE down and sigma projections and, with ``lm_head``, the LM head
    (the token embedding keeps its own table).  The dense weights are dropped.  Routers, gates of
    the depth engine, norms and the M-CMoE bases stay as they are; so does a weight whose input
    width is not a multiple of 32, or a head width that the fused prologue does not tile."""
    from .cham_memory import ContinuousHolographicMemory
    from .mcmoe import ManifoldContinuousMoE, SiTUGLU
    from .sssd_attention import SSSDAttention

    def pack(weights, pad=1):
        w = torch.cat([x.weight.detach() for x in weights], 0)
        if pad > 1 and w.shape[0] % pad:
            w = torch.cat([w, w.new_zeros(-w.shape[0] % pad, w.shape[1])], 0)
        return Int4Linear.from_weight(w, None, group_size, symmetric)

    def replace(owner, name):
        lin = getattr(owner, name)
        if isinstance(lin, nn.Linear) and lin.in_features % 32 == 0:
            setattr(owner, name, Int4Linear.from_linear(lin, group_size, symmetric))

    for m in list(model.modules()):
        if isinstance(m, SSSDAttention) and m.int4_in is None and m.hidden_dim % 32 == 0 and m.head_dim % 8 == 0:
            m.int4_in = pack([m.w_q, m.w_k, m.w_v, m.w_delta], 8)
            m.w_q = m.w_k = m.w_v = m.w_delta = None
            m._verace_cat = None
            replace(m, "w_out")
        elif isinstance(m, ContinuousHolographicMemory) and m.int4_in is None and m.hidden_dim % 32 == 0 \
                and m.holographic_dim % 8 == 0:
            m.int4_in = pack([m.w_q, m.w_k, m.w_v, m.w_gamma], 8)
            m.w_q = m.w_k = m.w_v = m.w_gamma = None
            m._verace_cat = None
            replace(m, "w_out")
        elif isinstance(m, SiTUGLU) and m.int4_in is None and m.fp8_in is None and m.in_features % 32 == 0:
            m.int4_in = pack([m.w_gate, m.w_up])
            m.w_gate = m.w_up = None
            m._stacked = m._stacked_key = None
        elif isinstance(m, ManifoldContinuousMoE):
            replace(m, "base_w_down")
            replace(m, "hyper_sigma")
    if lm_head and isinstance(getattr(model, "lm_head", None), nn.Linear):
        replace(model, "lm_head")
    return model
