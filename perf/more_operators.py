"""Cases of the feed-forward sub-layer's operators: the RMS norm (with the residual's addition)
whose output is in 8 bits with a scale a row, the gated block (both projections, the activation
and the product) with its backward pass, and the product with bias, activation and residual in
its epilogue, with its backward pass.

``run`` computes each of them either in its plain form (``own`` false: elementary torch
operations in 32 bits, one rounding at the end) or through the package (``own`` true).

The operators:

* norm: h <- h + y (where y is given; rounded to h's type), n = h / sqrt(mean h^2 + eps) w,
  a = max(max |n|, 2^-100) of the row; scale = a / 448, q = n 448 / a rounded to e4m3.
* gated: g = x Wgᵀ, u = x Wuᵀ, out = act(g) up(u); "situ": act(g) = b1 tanh(g / b1) sigmoid(g),
  up(u) = b2 tanh(u / b2); "silu", "gelu": that of g, up(u) = u.
  Backward, from the gradient d of out: dg = d act'(g) up(u), du = d act(g) up'(u),
  dx = dg Wg + du Wu, dWg = dgᵀ x, dWu = duᵀ x.
* linear: out = act(x Wᵀ + bias) + residual.  Backward, from d: p = d act'(x Wᵀ + bias),
  dx = p W, dW = pᵀ x, dbias = the sum of p over the rows, dresidual = d.

Operands in 8 bits are e4m3 with a scale in 32 bits for each row of x and of the weights.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1}
_E4M3 = torch.float8_e4m3fn
_package = None


def _own():
    """The package (its folder's name is no identifier), loaded at the first call."""
    global _package
    if _package is None:
        name = "verace_v1_b200"
        if name not in sys.modules:
            folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "verace-v1_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                          submodule_search_locations=[folder])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _package = sys.modules[name]
    return _package


# ---------------------------------------------------------------------------- the cases
def _norm(name, rows, cols, dtype, add=True):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "add": add}


def _gated(name, m, k, f, dtype, act="situ", train=False):
    return {"name": name, "op": "gated", "m": m, "k": k, "f": f, "dtype": dtype, "act": act, "train": train}


def _linear(name, m, k, n, dtype, act="", bias=False, residual=False, train=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "train": train}


def listed():
    return [
        # the norm ahead of the feed-forward block for one sequence's token: latency
        _norm("norm to 8 bits, one token", 1, 1024, "bf16"),
        # the same for a prompt of 16384 tokens at hidden 4096: bandwidth
        _norm("norm to 8 bits, 16384 tokens", 16384, 4096, "bf16"),
        # fp32 rows of a width that no vector divides, without a residual
        _norm("norm to 8 bits, fp32 ragged", 1111, 5001, "f32", add=False),
        # the feed-forward block of one decode step of one sequence, hidden 1024: latency
        _gated("gated, one token", 1, 1024, 2048, "bf16"),
        # a decode batch of 64 in 8 bits at hidden 4096: the weights' bytes
        _gated("gated, 64 tokens, 8 bits", 64, 4096, 8192, "fp8"),
        # a prompt's feed-forward block at hidden 4096
        _gated("gated, 8192 tokens", 8192, 4096, 8192, "bf16"),
        # a training step's, forward and backward
        _gated("gated training, 4096 tokens", 4096, 4096, 8192, "bf16", train=True),
        # training in fp32 over sizes that no tile divides
        _gated("gated training, fp32 ragged", 777, 1001, 2050, "f32", act="silu", train=True),
        # the down projection of a few sequences' decode step, with the residual
        _linear("linear down projection, 7 tokens", 7, 8192, 4096, "f16", bias=True, residual=True),
        # a prompt's down projection in 8 bits, with the residual
        _linear("linear, 8192 tokens, 8 bits", 8192, 8192, 4096, "fp8", residual=True),
        # a biased layer with an activation and a residual, forward and backward
        _linear("linear training, 2048 tokens", 2048, 4096, 4096, "bf16", "gelu", bias=True, residual=True, train=True),
        # fp16 over sizes that no tile and no vector divides
        _linear("linear ragged", 333, 1001, 5003, "f16", "silu", bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gated", "gated", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32", "fp8"])
    if op == "norm":
        rows = _log(rng, 1, 65536)
        cols = min(_log(rng, 64, 16384), (16384 * 4096) // rows)
        if rng.random() < 0.6:
            cols = -(-cols // 8) * 8
        c = _norm("", rows, cols, "bf16" if dtype == "fp8" else dtype, rng.random() < 0.7)
        del c["name"]
        return c
    train = dtype != "fp8" and rng.random() < 0.4
    m = _log(rng, 1, 8192)
    k, f = _log(rng, 64, 8192), _log(rng, 64, 16384)
    if rng.random() < 0.7:
        k, f = -(-k // 16) * 16, -(-f // 16) * 16
    # at most a quarter of the largest listed case's products, of fp32 a sixteenth
    most = 4096 * 4096 * 8192 * 6 // (4 * (3 if train else 1) * (2 if op == "gated" else 1) * (4 if dtype == "f32" else 1))
    m = max(1, min(m, most // (k * f)))
    if op == "gated":
        c = _gated("", m, k, f, dtype, rng.choice(["situ", "situ", "silu", "gelu"]), train)
    else:
        # no relu in training: a sum next to its border has either slope
        c = _linear("", m, k, f, dtype, rng.choice(["", "silu", "gelu"] if train else ["", "relu", "silu", "gelu"]),
                    rng.random() < 0.5, rng.random() < 0.5, train)
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"norm": _prepare_norm, "gated": _prepare_gated, "linear": _prepare_linear}[case["op"]](case, g)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _in_8_bits(t):
    """(e4m3 values, a scale for each row) of t."""
    s = t.abs().amax(1, keepdim=True) / 448
    return (t / s).to(_E4M3), s[:, 0].contiguous()


def _prepare_norm(c, g):
    rows, cols, dt = c["rows"], c["cols"], _DT[c["dtype"]]
    # a residual stream: rows of different size, a few channels that stand out
    h = _randn(g, rows, cols) * (0.5 + 3 * torch.rand(rows, 1, device="cuda", generator=g))
    h = h * torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 12.0, 1.0)
    norm = torch.nn.RMSNorm(cols, eps=1e-6, device="cuda", dtype=dt).requires_grad_(False)
    norm.weight.copy_(1 + 0.2 * _randn(g, cols))
    return {"op": "norm", "h": h.to(dt), "y": _randn(g, rows, cols).to(dt) if c["add"] else None, "norm": norm,
            "sum": torch.empty(rows, cols, dtype=dt, device="cuda") if c["add"] else None}


def _prepare_gated(c, g):
    m, k, f = c["m"], c["k"], c["f"]
    x, wg, wu = _randn(g, m, k), 2 * _randn(g, f, k) / math.sqrt(k), 2 * _randn(g, f, k) / math.sqrt(k)
    s = {"op": "gated", "act": c["act"], "train": c["train"], "dtype": torch.bfloat16, "sx": None, "sg": None,
         "su": None, "d": None}
    if c["dtype"] == "fp8":
        (s["x"], s["sx"]), (s["wg"], s["sg"]), (s["wu"], s["su"]) = _in_8_bits(x), _in_8_bits(wg), _in_8_bits(wu)
    else:
        s["dtype"] = dt = _DT[c["dtype"]]
        s["x"], s["wg"], s["wu"] = x.to(dt), wg.to(dt), wu.to(dt)
        if c["train"]:
            s["d"] = _randn(g, m, f).to(dt)
    return s


def _prepare_linear(c, g):
    m, k, n = c["m"], c["k"], c["n"]
    x, w = _randn(g, m, k), _randn(g, n, k) / math.sqrt(k)
    s = {"op": "linear", "act": c["act"] or None, "train": c["train"], "dtype": torch.bfloat16, "sx": None, "sw": None,
         "d": None}
    if c["dtype"] == "fp8":
        (s["x"], s["sx"]), (s["w"], s["sw"]) = _in_8_bits(x), _in_8_bits(w)
    else:
        s["dtype"] = _DT[c["dtype"]]
        s["x"], s["w"] = x.to(s["dtype"]), w.to(s["dtype"])
    s["bias"] = (0.5 * _randn(g, n)).to(s["dtype"]) if c["bias"] else None
    s["residual"] = _randn(g, m, n).to(s["dtype"]) if c["residual"] else None
    if c["train"]:
        s["d"] = _randn(g, m, n).to(s["dtype"])
    return s


# ---------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        V = _package or _own()
        if op == "norm":
            if s["y"] is None:
                return V.rmsnorm_fp8(s["h"], s["norm"])
            return (s["sum"],) + V.add_rmsnorm_fp8(s["h"], s["y"], s["norm"], out=s["sum"])
        if op == "gated":
            if not s["train"]:
                return V.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"], x_scale=s["sx"],
                                      gate_scale=s["sg"], up_scale=s["su"])
            leaves = [s[k].detach().requires_grad_() for k in ("x", "wg", "wu")]
            out = V.gated_linear(*leaves, activation=s["act"])
            return (out.detach(),) + torch.autograd.grad(out, leaves, s["d"])
        if not s["train"]:
            return V.fused_linear(s["x"], s["w"], s["bias"], activation=s["act"], residual=s["residual"],
                                  x_scale=s["sx"], w_scale=s["sw"])
        leaves = {k: s[k].detach().requires_grad_() for k in ("x", "w", "bias", "residual") if s[k] is not None}
        out = V.fused_linear(leaves["x"], leaves["w"], leaves.get("bias"), activation=s["act"],
                             residual=leaves.get("residual"))
        return (out.detach(),) + torch.autograd.grad(out, list(leaves.values()), s["d"])
    return {"norm": _plain_norm, "gated": _plain_gated, "linear": _plain_linear}[op](s)


def _plain_norm(s):
    h, norm = s["h"], s["norm"]
    if s["y"] is not None:
        h = (h.float() + s["y"].float()).to(h.dtype)
    n = h.float()
    n = n * torch.rsqrt(n.square().mean(1, keepdim=True) + norm.eps) * norm.weight.float()
    top = n.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    q = (n * (448 / top)).to(_E4M3), (top / 448)[:, 0]
    return q if s["y"] is None else (h,) + q


def _act(name, z, want_slope):
    """act(z), and its derivative where it is asked for."""
    if name is None:
        return z, torch.ones_like(z) if want_slope else None
    if name == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).float() if want_slope else None
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p)) if want_slope else None
    half = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))        # gelu: z times the normal distribution's share below z
    return z * half, half + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi) if want_slope else None


def _gates(s, g, u, want_slope):
    """act(g), up(u), and their derivatives."""
    if s["act"] != "situ":
        a, da = _act(s["act"], g, want_slope)
        return a, u, da, torch.ones_like(u) if want_slope else None
    tg, tu, p = torch.tanh(g / 4.0), torch.tanh(u / 25.0), 1 / (1 + torch.exp(-g))
    a, b = 4.0 * tg * p, 25.0 * tu
    if not want_slope:
        return a, b, None, None
    return a, b, (1 - tg * tg) * p + 4.0 * tg * p * (1 - p), 1 - tu * tu


def _wide(t, scale):
    return t.float() if scale is None else t.float() * scale[:, None]


def _plain_gated(s):
    dt = s["dtype"]
    x, wg, wu = _wide(s["x"], s["sx"]), _wide(s["wg"], s["sg"]), _wide(s["wu"], s["su"])
    g, u = x @ wg.t(), x @ wu.t()
    a, b, da, db = _gates(s, g, u, s["train"])
    if not s["train"]:
        return (a * b).to(dt)
    d = s["d"].float()
    dg, du = d * da * b, d * a * db
    return (a * b).to(dt), (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)


def _plain_linear(s):
    dt = s["dtype"]
    x, w = _wide(s["x"], s["sx"]), _wide(s["w"], s["sw"])
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _act(s["act"], z, s["train"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["train"]:
        return y.to(dt)
    p = s["d"].float() * slope
    out = [y.to(dt), (p @ w).to(dt), (p.t() @ x).to(dt)]
    if s["bias"] is not None:
        out.append(p.sum(0).to(dt))
    if s["residual"] is not None:
        out.append(s["d"])
    return tuple(out)


# ---------------------------------------------------------------------------- the floor
def work(c):
    e = _SIZE[c["dtype"]]
    if c["op"] == "norm":
        rows, cols = c["rows"], c["cols"]
        return {"bytes": rows * cols * (e * (3 if c["add"] else 1) + 1) + cols * e + 4 * rows, "flops": 6 * rows * cols}
    m, k, o = c["m"], c["k"], 2 if c["dtype"] == "fp8" else e
    scaled = 4 if c["dtype"] == "fp8" else 0
    if c["op"] == "gated":
        f = c["f"]
        size = e * (m * k + 2 * f * k) + o * m * f + scaled * (m + 2 * f)
        if not c["train"]:
            return {"bytes": size, "flops": 4 * m * k * f}
        return {"bytes": size + e * (m * f + m * k + 2 * f * k), "flops": 12 * m * k * f}
    n = c["n"]
    size = e * (m * k + n * k) + o * (m * n * (2 if c["residual"] else 1) + (n if c["bias"] else 0)) + scaled * (m + n)
    if not c["train"]:
        return {"bytes": size, "flops": 2 * m * k * n}
    return {"bytes": size + e * (m * n + m * k + n * k + (n if c["bias"] else 0)), "flops": 6 * m * k * n}


# ---------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "gated": _exact_gated, "linear": _exact_linear}[case["op"]](s)


def _exact_norm(s):
    h = s["h"].double()
    if s["y"] is not None:
        h = (h + s["y"].double()).to(s["h"].dtype).double()
    n = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + s["norm"].eps).sqrt() * s["norm"].weight.double()
    scale = torch.clamp(n.abs().max(1, keepdim=True).values, min=2.0 ** -100) / 448
    q = n / scale, scale[:, 0]
    return q if s["y"] is None else (h,) + q


def _in_64(t, scale):
    return t.double() if scale is None else t.double() * scale.double()[:, None]


def _exact_act(name, z):
    if name is None:
        return z
    return {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[name](z)


def _gradients(out, leaves, d):
    return tuple(torch.autograd.grad(out, leaves, d.double()))


def _exact_gated(s):
    leaves = [_in_64(s[a], s[b]).requires_grad_(s["train"]) for a, b in (("x", "sx"), ("wg", "sg"), ("wu", "su"))]
    x, wg, wu = leaves
    g, u = torch.nn.functional.linear(x, wg), torch.nn.functional.linear(x, wu)
    if s["act"] == "situ":
        out = 4 * torch.tanh(g / 4) * torch.sigmoid(g) * (25 * torch.tanh(u / 25))
    else:
        out = _exact_act(s["act"], g) * u
    if not s["train"]:
        return out
    return (out.detach(),) + _gradients(out, leaves, s["d"])


def _exact_linear(s):
    leaves = {"x": _in_64(s["x"], s["sx"]), "w": _in_64(s["w"], s["sw"])}
    for k in ("bias", "residual"):
        if s[k] is not None:
            leaves[k] = s[k].double()
    for t in leaves.values():
        t.requires_grad_(s["train"])
    out = _exact_act(s["act"], torch.nn.functional.linear(leaves["x"], leaves["w"], leaves.get("bias")))
    if "residual" in leaves:
        out = out + leaves["residual"]
    if not s["train"]:
        return out
    return (out.detach(),) + _gradients(out, list(leaves.values()), s["d"])
