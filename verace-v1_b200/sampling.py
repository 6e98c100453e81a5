"""From logits to tokens at the end of a decode step: penalties, biases and grammar masks
(``verace_logits_process``), and the choice of a token (``verace_sample``).

The reference's generator takes the arg-max of the raw logits
(verace_v1/serving/hyper_generate.py:58-77); ``sample_logits(logits, temperature=0)`` is
that choice.  All controls may differ per row of the batch: a number holds for every row, a
[b] tensor for each its own.  Nothing here synchronises with the host.
"""
from typing import Optional, Tuple, Union

import torch

from ._lib import F32, check, lib
from ._launch import current, raw_stream, wrote
from .int4 import _require_no_grad
from .kernels import _DTYPE

PerRow = Union[float, torch.Tensor]
_INF = float("inf")


_INT32 = torch.iinfo(torch.int32)


def _int32(value: torch.Tensor) -> torch.Tensor:
    """value as int32; an int64 one beyond its range (a limit that is meant to hold nothing back) as its end."""
    if value.dtype is torch.int64:
        value = value.clamp(_INT32.min, _INT32.max)
    return value.to(torch.int32)


def _per_row(value: torch.Tensor, name: str, b: int, dev, dtype=torch.float32) -> torch.Tensor:
    assert value.dim() == 1 and value.shape[0] == b and value.device == dev, \
        f"{name} must be a number or a [b] tensor on the logits' device"
    if value.dtype is not dtype or not value.is_contiguous():
        value = (_int32(value) if dtype is torch.int32 else value.to(dtype)).contiguous()
    return value


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
    return lengths if lengths.dtype is torch.int32 and lengths.is_contiguous() else _int32(lengths).contiguous()


def _dense_rows(x: torch.Tensor, b: int, v: int) -> int:
    """The row stride of x [b, v], or 0 where its rows are not dense and apart."""
    if v > 1 and x.stride(1) != 1:
        return 0
    if b <= 1:
        return max(v, 1)
    ld = x.stride(0)
    return ld if ld >= v else 0


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
    assert logits.is_cuda, "This kernel requires CUDA tensors"
    assert logits.dim() == 2, "logits must be [b, v]"
    if logits.requires_grad:
        _require_no_grad(logits, "process_logits")
    dev = logits.device
    index = dev.index
    if index != current():
        with torch.cuda.device(dev):
            return process_logits(logits, tokens, lengths, prompt_lengths, repetition_penalty=repetition_penalty,
                                  presence_penalty=presence_penalty, frequency_penalty=frequency_penalty,
                                  bias_ids=bias_ids, bias_values=bias_values, allowed=allowed, out=out,
                                  out_dtype=out_dtype)
    dt = logits.dtype
    code = _DTYPE.get(dt)
    if code is None:
        raise ValueError(f"process_logits: {dt} logits (expected fp32, bf16 or fp16)")
    b, v = logits.shape
    ld = _dense_rows(logits, b, v)
    if not ld:
        assert out is not logits, "in-place processing needs dense rows"
        logits, ld = logits.contiguous(), max(v, 1)
    given = out is not None
    if not given:
        if out_dtype is None or out_dtype is dt:
            out, ocode = logits.new_empty((b, v)), code
        elif out_dtype is torch.float32:
            out, ocode = logits.new_empty((b, v), dtype=out_dtype), F32
        else:
            raise ValueError(f"process_logits: out_dtype {out_dtype} (expected {dt} or torch.float32)")
        old = max(v, 1)
    else:
        old = _dense_rows(out, b, v) if out.shape == logits.shape else 0
        assert old and out.device == dev and out.dtype in (dt, torch.float32) and out_dtype in (None, out.dtype), \
            "out must be [b, v] with dense rows, in the logits' dtype or fp32"
        ocode = _DTYPE[out.dtype]
    rp = pp = fp = None
    rs = ps = fs = 0.0
    if isinstance(repetition_penalty, torch.Tensor):
        repetition_penalty = _per_row(repetition_penalty, "repetition_penalty", b, dev)
        rp = repetition_penalty.data_ptr()
    elif repetition_penalty > 0:
        rs = repetition_penalty
    else:
        raise ValueError(f"repetition_penalty {repetition_penalty}: expected a number above 0")
    if isinstance(presence_penalty, torch.Tensor):
        presence_penalty = _per_row(presence_penalty, "presence_penalty", b, dev)
        pp = presence_penalty.data_ptr()
    else:
        ps = presence_penalty
    if isinstance(frequency_penalty, torch.Tensor):
        frequency_penalty = _per_row(frequency_penalty, "frequency_penalty", b, dev)
        fp = frequency_penalty.data_ptr()
    else:
        fs = frequency_penalty
    tp = lp = qp = None
    tld = t64 = L = 0
    if tokens is not None:
        assert tokens.dim() == 2 and tokens.shape[0] == b and tokens.device == dev, \
            "tokens must be [b, L] on the logits' device"
        t64 = _ids(tokens, "tokens")
        L = tokens.shape[1]
        tld = _dense_rows(tokens, b, L)
        if not tld:
            tokens, tld = tokens.contiguous(), max(L, 1)
        tp = tokens.data_ptr()
        if lengths is not None:
            lengths = _lengths(lengths, "lengths", b, dev)
            lp = lengths.data_ptr()
        if prompt_lengths is not None:
            prompt_lengths = _lengths(prompt_lengths, "prompt_lengths", b, dev)
            qp = prompt_lengths.data_ptr()
    ip = vp = None
    nb = b64 = 0
    if bias_ids is not None or bias_values is not None:
        assert bias_ids is not None and bias_values is not None, "bias_ids and bias_values go together"
        assert bias_ids.dim() == 2 and bias_ids.shape[0] == b and bias_values.shape == bias_ids.shape \
            and bias_ids.device == dev and bias_values.device == dev, "bias_ids and bias_values must be [b, n]"
        b64 = _ids(bias_ids, "bias_ids")
        nb = bias_ids.shape[1]
        bias_ids = bias_ids.contiguous()
        bias_values = bias_values.float().contiguous()
        if nb:
            ip, vp = bias_ids.data_ptr(), bias_values.data_ptr()
    ap, ald = None, 0
    if allowed is not None:
        words = (v + 31) // 32
        rows = allowed.shape[0]
        assert allowed.dtype is torch.int32 and allowed.shape == (rows, words) and rows in (1, b) \
            and allowed.device == dev, "allowed must be int32 [b or 1, ceil(v / 32)] on the logits' device"
        ald = _dense_rows(allowed, rows, words)
        if not ald:
            allowed, ald = allowed.contiguous(), words
        if rows == 1:
            ald = 0
        ap = allowed.data_ptr()
    rc = lib().verace_logits_process(logits.data_ptr(), ld, out.data_ptr(), old, b, v, code, ocode, tp, tld, t64, L, lp,
                                     qp, rp, rs, pp, ps, fp, fs, ip, vp, nb, b64, ap, ald, raw_stream(index))
    if rc:
        check(rc, "verace_logits_process")
    if given:
        wrote(out)
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
    assert logits.is_cuda, "This kernel requires CUDA tensors"
    assert logits.dim() == 2, "logits must be [b, v]"
    if logits.requires_grad:
        _require_no_grad(logits, "sample_logits")
    dev = logits.device
    index = dev.index
    if index != current():
        with torch.cuda.device(dev):
            return sample_logits(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    code = _DTYPE.get(logits.dtype)
    if code is None:
        raise ValueError(f"sample_logits: {logits.dtype} logits (expected fp32, bf16 or fp16)")
    b, v = logits.shape
    assert v > 0, "logits must have at least one column"
    tp = kp = pp = mp = None
    ts = ps = ms = 0.0
    ks = 0
    if isinstance(temperature, torch.Tensor):
        temperature = _per_row(temperature, "temperature", b, dev)
        tp = temperature.data_ptr()
    else:
        ts = temperature
        if not 0 <= ts < _INF:
            raise ValueError(f"temperature {ts}: expected a finite number of at least 0")
    if isinstance(top_k, torch.Tensor):
        top_k = _per_row(top_k, "top_k", b, dev, torch.int32)
        kp = top_k.data_ptr()
    else:
        ks = top_k if 0 < top_k < v else 0
    if isinstance(top_p, torch.Tensor):
        top_p = _per_row(top_p, "top_p", b, dev)
        pp = top_p.data_ptr()
    else:
        ps = top_p
    if isinstance(min_p, torch.Tensor):
        min_p = _per_row(min_p, "min_p", b, dev)
        mp = min_p.data_ptr()
    else:
        ms = min_p
    ld = _dense_rows(logits, b, v)
    if not ld:
        logits, ld = logits.contiguous(), v
    np_, nld = None, 0
    if tp is not None or ts > 0:
        if noise is None:
            raise ValueError("sample_logits: noise is needed unless temperature is 0")
        assert noise.dtype is torch.float32 and noise.shape == logits.shape and noise.device == dev, \
            "noise must be fp32 in the logits' shape"
        nld = _dense_rows(noise, b, v)
        if not nld:
            noise, nld = noise.contiguous(), v
        np_ = noise.data_ptr()
    tokens = logits.new_empty(b, dtype=torch.int64)
    logprobs = logits.new_empty(b, dtype=torch.float32)
    rc = lib().verace_sample(logits.data_ptr(), ld, np_, nld, b, v, code, tp, ts, kp, ks, pp, ps, mp, ms,
                             tokens.data_ptr(), logprobs.data_ptr(), raw_stream(index))
    if rc:
        check(rc, "verace_sample")
    return tokens, logprobs
