"""From logits to tokens at the end of a decode step: penalties, biases and grammar masks
(``verace_logits_process``), and the choice of a token (``verace_sample``).

The reference's generator takes the arg-max of the raw logits
(verace_v1/serving/hyper_generate.py:58-77); ``sample_logits(logits, temperature=0)`` is
that choice.  All controls may differ per row of the batch: a number holds for every row, a
[b] tensor for each its own.  Nothing here synchronises with the host.
"""
from typing import Optional, Tuple, Union

import torch

from ._lib import check, lib
from ._launch import launch
from .int4 import _require_no_grad
from .kernels import _DTYPE

PerRow = Union[float, torch.Tensor]


def _per_row(value: PerRow, name: str, b: int, dev, dtype=torch.float32):
    """(tensor or None, its pointer or None, the scalar beside it)"""
    if not isinstance(value, torch.Tensor):
        return None, None, value
    assert value.dim() == 1 and value.shape[0] == b and value.device == dev, \
        f"{name} must be a number or a [b] tensor on the logits' device"
    if value.dtype is not dtype or not value.is_contiguous():
        value = value.to(dtype).contiguous()
    return value, value.data_ptr(), 0


def _ids(ids: torch.Tensor, name: str):
    if ids.dtype is torch.int64:
        return 1
    assert ids.dtype is torch.int32, f"{name} must be int32 or int64"
    return 0


def _lengths(lengths: Optional[torch.Tensor], name: str, b: int, dev):
    if lengths is None:
        return None
    assert lengths.dim() == 1 and lengths.shape[0] == b and lengths.device == dev, \
        f"{name} must be a [b] tensor on the logits' device"
    return lengths if lengths.dtype is torch.int32 and lengths.is_contiguous() else lengths.to(torch.int32).contiguous()


def _logit_rows(logits: torch.Tensor, who: str) -> torch.Tensor:
    assert logits.is_cuda, "This kernel requires CUDA tensors"
    assert logits.dim() == 2, "logits must be [b, v]"
    _require_no_grad(logits, who)
    if logits.dtype not in _DTYPE:
        raise ValueError(f"{who}: {logits.dtype} logits (expected fp32, bf16 or fp16)")
    return logits


def _row_stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def process_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None, *,
                   repetition_penalty: PerRow = 1.0, presence_penalty: PerRow = 0.0, frequency_penalty: PerRow = 0.0,
                   bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """logits [b, v] (fp32, bf16 or fp16; any row stride) with, in this order and in fp32:

    * l / r for l > 0, else l * r, r = ``repetition_penalty`` (above 0), where the token occurs
      in the row's history;
    * l - ``frequency_penalty`` * c - ``presence_penalty`` where it occurs c > 0 times among the
      generated tokens;
    * l + value for the row's ``bias_ids`` / ``bias_values`` [b, n]; the last of equal ids holds;
    * -inf where ``allowed`` has a 0 bit: int32 [b or 1, ceil(v / 32)], token t in bit t % 32 of
      word t // 32.

    The history is ``tokens`` [b, L] (int32 or int64), row i's first ``lengths[i]`` of them (all
    by default), the first ``prompt_lengths[i]`` (none by default) being the prompt.  Ids outside
    [0, v) are skipped, so lists may be padded with -1.  Returns a new tensor in the logits' dtype
    or ``out_dtype`` (fp32), or ``out`` (which may be ``logits`` itself)."""
    _logit_rows(logits, "process_logits")
    dev, dt = logits.device, logits.dtype
    b, v = logits.shape
    if v > 1 and logits.stride(1) != 1 or b > 1 and logits.stride(0) < v:
        assert out is not logits, "in-place processing needs dense rows"
        logits = logits.contiguous()
    if out is None:
        odt = dt if out_dtype is None else out_dtype
        if odt is not dt and odt is not torch.float32:
            raise ValueError(f"process_logits: out_dtype {odt} (expected {dt} or torch.float32)")
        out = torch.empty((b, v), dtype=odt, device=dev)
    else:
        odt = out.dtype
        assert out.shape == logits.shape and out.device == dev and (v <= 1 or out.stride(1) == 1) \
            and odt in (dt, torch.float32) and out_dtype in (None, odt) and (b <= 1 or out.stride(0) >= v), \
            "out must be [b, v] with dense rows, in the logits' dtype or fp32"
    if not isinstance(repetition_penalty, torch.Tensor) and not repetition_penalty > 0:
        raise ValueError(f"repetition_penalty {repetition_penalty}: expected a number above 0")
    rt, rp, rs = _per_row(repetition_penalty, "repetition_penalty", b, dev)
    pt, pp, ps = _per_row(presence_penalty, "presence_penalty", b, dev)
    ft, fp, fs = _per_row(frequency_penalty, "frequency_penalty", b, dev)
    tp, tld, t64, L = None, 0, 0, 0
    if tokens is not None:
        assert tokens.dim() == 2 and tokens.shape[0] == b and tokens.device == dev, \
            "tokens must be [b, L] on the logits' device"
        t64 = _ids(tokens, "tokens")
        L = tokens.shape[1]
        if L > 1 and tokens.stride(1) != 1 or b > 1 and tokens.stride(0) < L:
            tokens = tokens.contiguous()
        tp, tld = tokens.data_ptr(), tokens.stride(0) if b > 1 else L
    lengths = _lengths(lengths, "lengths", b, dev)
    prompt_lengths = _lengths(prompt_lengths, "prompt_lengths", b, dev)
    nb, b64 = 0, 0
    assert (bias_ids is None) == (bias_values is None), "bias_ids and bias_values go together"
    if bias_ids is not None:
        assert bias_ids.dim() == 2 and bias_ids.shape[0] == b and bias_values.shape == bias_ids.shape \
            and bias_ids.device == dev and bias_values.device == dev, "bias_ids and bias_values must be [b, n]"
        b64 = _ids(bias_ids, "bias_ids")
        nb = bias_ids.shape[1]
        bias_ids = bias_ids.contiguous()
        bias_values = bias_values.float().contiguous()
    ap, ald = None, 0
    if allowed is not None:
        words = (v + 31) // 32
        assert allowed.dtype is torch.int32 and allowed.dim() == 2 and allowed.shape[0] in (1, b) \
            and allowed.shape[1] == words and allowed.device == dev, \
            "allowed must be int32 [b or 1, ceil(v / 32)] on the logits' device"
        if words > 1 and allowed.stride(1) != 1 or allowed.shape[0] > 1 and allowed.stride(0) < words:
            allowed = allowed.contiguous()
        ap, ald = allowed.data_ptr(), allowed.stride(0) if allowed.shape[0] > 1 else 0
    rc = launch(dev, lib().verace_logits_process, logits.data_ptr(), _row_stride(logits), out.data_ptr(),
                _row_stride(out), b, v, _DTYPE[dt], _DTYPE[odt], tp, tld, t64, L,
                None if lengths is None else lengths.data_ptr(),
                None if prompt_lengths is None else prompt_lengths.data_ptr(), rp, rs, pp, ps, fp, fs,
                None if nb == 0 else bias_ids.data_ptr(), None if nb == 0 else bias_values.data_ptr(), nb, b64, ap,
                ald)
    if rc:
        check(rc, "verace_logits_process")
    return out


def sample_logits(logits: torch.Tensor, noise: Optional[torch.Tensor] = None, *, temperature: PerRow = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: PerRow = 1.0, min_p: PerRow = 0.0
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token per row of logits [b, v]: (tokens [b] int64, log-probabilities [b] fp32).

    With z = (logits - their largest) / temperature, kept are the tokens with z at least the ``top_k``-th largest
    (0: all), of those the ones with less than ``top_p`` of the kept mass strictly above them,
    and exp(z) >= ``min_p`` (the largest always is); equal values are kept or dropped together.  The token is
    the arg-max over the kept of z - log(noise), the lowest index on ties: with ``noise`` [b, v]
    fp32 drawn from Exp(1) (``torch.empty(b, v).exponential_()``) a draw from the softmax over
    the kept.  Temperature 0: the largest logit; no noise, no truncation.  The log-probability is
    log softmax(z) over the whole row (temperature 0: of the logits).  NaN and -inf are never
    chosen; a row with nothing else gives token -1 and -inf."""
    _logit_rows(logits, "sample_logits")
    dev = logits.device
    b, v = logits.shape
    assert v > 0, "logits must have at least one column"
    tt, tp, ts = _per_row(temperature, "temperature", b, dev)
    if tt is None and not 0 <= ts < float("inf"):
        raise ValueError(f"temperature {ts}: expected a finite number of at least 0")
    kt, kp, ks = _per_row(top_k, "top_k", b, dev, torch.int32)
    pt, pp, ps = _per_row(top_p, "top_p", b, dev)
    mt, mp, ms = _per_row(min_p, "min_p", b, dev)
    if v > 1 and logits.stride(1) != 1 or b > 1 and logits.stride(0) < v:
        logits = logits.contiguous()
    if tt is not None or ts > 0:
        if noise is None:
            raise ValueError("sample_logits: noise is needed unless temperature is 0")
        assert noise.dtype is torch.float32 and noise.shape == logits.shape and noise.device == dev, \
            "noise must be fp32 in the logits' shape"
        if v > 1 and noise.stride(1) != 1 or b > 1 and noise.stride(0) < v:
            noise = noise.contiguous()
    else:
        noise = None
    tokens = torch.empty(b, dtype=torch.int64, device=dev)
    logprobs = torch.empty(b, dtype=torch.float32, device=dev)
    rc = launch(dev, lib().verace_sample, logits.data_ptr(), _row_stride(logits),
                None if noise is None else noise.data_ptr(), 0 if noise is None else _row_stride(noise), b, v,
                _DTYPE[logits.dtype], tp, ts, kp, ks, pp, ps, mp, ms, tokens.data_ptr(), logprobs.data_ptr())
    if rc:
        check(rc, "verace_sample")
    return tokens, logprobs
