"""Cases of the operators at the end of a decode step: the product of a few tokens with 4-bit
weights, the processing of logits (penalties, biases, grammar masks) and the choice of a token.

``run`` computes each of them either in its plain form (``own`` false: elementary torch
operations in 32 bits, one rounding at the end) or through the package (``own`` true).

The operators:

* int4: y = x Wᵀ (+ bias), W[n, k] = s[k // G, n] (q[n, k] - z[k // G, n]); q in 4 bits,
  two to a byte along k (the even k in the low half), z = 8 where no zeros are given.
* process: per row of logits l, with c the counts of the generated tokens in the row's history
  and "seen" any token of it, the prompt's included:
  l <- l / r if l > 0 else l r (seen);  l <- l - f c - p [c > 0];  l <- l + bias;
  l <- -inf where the grammar's bit is 0.
* sample: z = l / T; kept are the tokens that are at least the k-th largest, that have less
  than p of the mass of those above them (mass among the k kept), and exp(z - max) >= min_p;
  token = argmax over the kept of z - log(noise), noise drawn from Exp(1) (T = 0: the largest
  logit, no noise); and log softmax(z) of it (T = 0: of l).
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_INF = float("inf")
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
def _int4(name, m, n, k, group, dtype, zeros=False, bias=False, out="same"):
    return {"name": name, "op": "int4", "m": m, "n": n, "k": k, "group": group, "dtype": dtype, "zeros": zeros,
            "bias": bias, "out": out}


def _process(name, b, v, length, dtype, pad=0, biases=0, mask=False, out="same"):
    return {"name": name, "op": "process", "b": b, "v": v, "length": length, "dtype": dtype, "pad": pad,
            "biases": biases, "mask": mask, "out": out}


def _sample(name, b, v, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, masked=0.0):
    return {"name": name, "op": "sample", "b": b, "v": v, "dtype": dtype, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "masked": masked}


def listed():
    return [
        # the q, k, v and gate projection of one decode step of one sequence, hidden 1024: latency
        _int4("int4 projection, one token", 1, 3080, 1024, 128, "bf16"),
        # the LM head over the default vocabulary for one sequence
        _int4("int4 LM head, one token", 1, 163840, 1024, 128, "bf16", zeros=True, out="f32"),
        # the down projection at hidden 4096 for a few sequences, finer groups, fp16
        _int4("int4 down projection, 7 tokens", 7, 4096, 8192, 64, "f16", zeros=True),
        # the gate/up projection at hidden 4096 for a decode batch of 64
        _int4("int4 gate/up, 64 tokens", 64, 16384, 4096, 128, "bf16"),
        # the gate/up projection at the modules' default width, 16 sequences: the largest
        _int4("int4 wide gate/up, 16 tokens", 16, 65536, 16384, 128, "bf16"),
        # a vocabulary with an added token, fp32, a width no tile divides, the finest groups
        _int4("int4 fp32 ragged, 5 tokens", 5, 32001, 1056, 32, "f32", zeros=True, bias=True),
        # one sequence's logits after a short prompt: latency
        _process("process, one row", 1, 32000, 200, "f32"),
        # a serving batch: ragged histories, biases, a grammar's mask; 16-bit logits widened
        _process("process, 64 rows, grammar", 64, 163840, 4096, "bf16", biases=300, mask=True, out="f32"),
        # a few rows with the history of a long document, rows of a padded vocabulary
        _process("process, long histories", 8, 32000, 65536, "bf16", pad=64, mask=True),
        # greedy choice for one sequence: latency
        _sample("sample, greedy, one row", 1, 32000, "f32", temperature=0.0),
        # a serving batch with every truncation, over masked logits
        _sample("sample, truncated, 64 rows", 64, 163840, "f32", 0.8, 50, 0.9, 0.02, masked=0.3),
        # many rows of untruncated sampling (rollouts)
        _sample("sample, untruncated, 256 rows", 256, 32000, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int4", "int4", "process", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "int4":
        m = _log(rng, 1, 64)
        k = 32 * _log(rng, 8, 512)
        n = min(_log(rng, 64, 163840), (1 << 30) // (k * -(-m // 16)))
        c = _int4("", m, n, k, rng.choice([32, 64, 128, 128]), dtype, rng.random() < 0.5, rng.random() < 0.3,
                  rng.choice(["same", "same", "f32"]))
    elif op == "process":
        b = _log(rng, 1, 128)
        v = min(_log(rng, 1000, 163840), 64 * 163840 // b)
        length = min(_log(rng, 1, 65536), (1 << 19) // b)
        c = _process("", b, v, length, dtype, rng.choice([0, 0, 3, 64]), rng.choice([0, 0, 17, 300]),
                     rng.random() < 0.5, rng.choice(["same", "f32"]))
    else:
        b = _log(rng, 1, 256)
        v = min(_log(rng, 1000, 163840), 64 * 163840 // b)
        c = _sample("", b, v, dtype, rng.choice([0.0, 0.7, 1.0, 1.3]), rng.choice([0, 0, 1, 20, 50, 1000]),
                    rng.choice([1.0, 1.0, 0.9, 0.5]), rng.choice([0.0, 0.0, 0.05]), rng.choice([0.0, 0.5, 0.99]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"int4": _prepare_int4, "process": _prepare_process, "sample": _prepare_sample}[case["op"]](case, g)


def _prepare_int4(c, g):
    m, n, k, group = c["m"], c["n"], c["k"], c["group"]
    dt = _DT[c["dtype"]]
    groups = -(-k // group)
    q = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    rows = max(1, (1 << 26) // k)
    for i in range(0, n, rows):     # bell-shaped codes, as quantised weights have them
        part = torch.randn(min(rows, n - i), k, device="cuda", generator=g).mul_(2.6).add_(8).round_().clamp_(0, 15)
        part = part.to(torch.uint8)
        q[i:i + rows] = part[:, 0::2] | (part[:, 1::2] << 4)
    scales = (0.3 + 0.2 * torch.rand(groups, n, device="cuda", generator=g)) / math.sqrt(k)
    zeros = torch.randint(6, 11, (groups, n), device="cuda", generator=g, dtype=torch.uint8) if c["zeros"] else None
    bias = (0.1 * torch.randn(n, device="cuda", generator=g)).to(dt) if c["bias"] else None
    return {"op": "int4", "x": torch.randn(m, k, device="cuda", generator=g).to(dt), "q": q, "s": scales.to(dt),
            "z": zeros, "bias": bias, "group": group, "out": torch.float32 if c["out"] == "f32" else dt}


def _prepare_process(c, g):
    b, v, length = c["b"], c["v"], c["length"]
    dt = _DT[c["dtype"]]
    logits = (3 * torch.randn(b, v + c["pad"], device="cuda", generator=g)).to(dt)[:, :v]
    # token frequencies as in text: log-uniform ranks; each row's list is filled to a length of its own
    u = torch.rand(b, length, device="cuda", generator=g)
    tokens = (torch.exp(u * math.log(v)) - 1).long().clamp_(0, v - 1) * 7919 % v
    lengths = (length * (0.3 + 0.7 * torch.rand(b, device="cuda", generator=g))).int()
    lengths[0] = length
    prompt = (lengths * torch.rand(b, device="cuda", generator=g)).int()
    s = {"op": "process", "logits": logits, "tokens": tokens, "lengths": lengths, "prompt": prompt,
         "r": 1 + 0.3 * torch.rand(b, device="cuda", generator=g), "p": 0.5 * torch.rand(b, device="cuda", generator=g),
         "f": 0.2 * torch.rand(b, device="cuda", generator=g), "ids": None, "values": None, "mask": None,
         "out": torch.float32 if c["out"] == "f32" else dt}
    if c["biases"]:
        n = min(c["biases"], v)
        s["ids"] = torch.rand(b, v, device="cuda", generator=g).topk(n, dim=1).indices
        s["ids"][:, n - 1] = -1     # a padded list
        s["values"] = 4 * torch.randn(b, n, device="cuda", generator=g)
    if c["mask"]:                   # some rows free, some left with few tokens
        words = torch.randint(-2**31, 2**31, (b, -(-v // 32)), device="cuda", generator=g).int()
        few = torch.randint(-2**31, 2**31, words.shape, device="cuda", generator=g).int()
        words = torch.where(torch.arange(b, device="cuda")[:, None] % 3 == 0, words & few & (few >> 7), words)
        words[1::3] = -1
        s["mask"] = words
    return s


def _prepare_sample(c, g):
    b, v = c["b"], c["v"]
    logits = 2.5 * torch.randn(b, v, device="cuda", generator=g)
    if c["masked"]:
        logits = logits.masked_fill(torch.rand(b, v, device="cuda", generator=g) < c["masked"], -_INF)
    s = {"op": "sample", "logits": logits.to(_DT[c["dtype"]]), "noise": None, "t": c["temperature"],
         "top_k": c["top_k"], "top_p": c["top_p"], "min_p": c["min_p"]}
    if c["temperature"] > 0:
        s["noise"] = torch.empty(b, v, device="cuda").exponential_(generator=g)
    return s


# ---------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if own:
        V = _package or _own()
        if op == "int4":
            return V.int4_linear(s["x"], s["q"], s["s"], s["z"], s["bias"], group_size=s["group"], out_dtype=s["out"])
        if op == "process":
            return V.process_logits(s["logits"], s["tokens"], s["lengths"], s["prompt"], repetition_penalty=s["r"],
                                    presence_penalty=s["p"], frequency_penalty=s["f"], bias_ids=s["ids"],
                                    bias_values=s["values"], allowed=s["mask"], out_dtype=s["out"])
        return V.sample_logits(s["logits"], s["noise"], temperature=s["t"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"])
    return {"int4": _plain_int4, "process": _plain_process, "sample": _plain_sample}[op](s)


def _plain_int4(s):
    q, k = s["q"], s["x"].shape[1]
    codes = torch.stack((q & 15, q >> 4), dim=-1).view(q.shape[0], k).float()
    of_k = torch.arange(k, device=q.device) // s["group"]
    zero = 8.0 if s["z"] is None else s["z"].float().t()[:, of_k]
    y = s["x"].float() @ ((codes - zero) * s["s"].float().t()[:, of_k]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"])


def _plain_process(s):
    x = s["logits"].float()
    b, v = x.shape
    tokens = s["tokens"]
    at = torch.arange(tokens.shape[1], device=x.device)
    valid = (at < s["lengths"][:, None]) & (tokens >= 0) & (tokens < v)
    made = valid & (at >= s["prompt"][:, None])
    count = torch.zeros(2, b, v + 1, dtype=torch.int32, device=x.device)
    one = torch.ones_like(tokens, dtype=torch.int32)
    count[0].scatter_add_(1, torch.where(valid, tokens, v), one)
    count[1].scatter_add_(1, torch.where(made, tokens, v), one)
    seen, c = count[0, :, :v] > 0, count[1, :, :v].float()
    r = s["r"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["f"][:, None] * c - s["p"][:, None] * (c > 0)
    if s["ids"] is not None:
        ids = torch.where((s["ids"] >= 0) & (s["ids"] < v), s["ids"], v)
        x = x + torch.zeros(b, v + 1, device=x.device).scatter_(1, ids, s["values"])[:, :v]
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.view(b, -1)[:, :v] == 1, x, -_INF)
    return x.to(s["out"])


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), -_INF, x)
    b, v = x.shape
    z = x / s["t"] if s["t"] > 0 else x
    top = z.amax(1, keepdim=True)
    w = torch.where(z == top, 1.0, torch.exp(z - top))
    w = torch.where(top == -_INF, 0.0, w)
    total = w.sum(1, keepdim=True)
    if s["t"] > 0:
        keep = z > -_INF
        if 0 < s["top_k"] < v or s["top_p"] < 1:
            down, order = z.sort(dim=1, descending=True)
            if 0 < s["top_k"] < v:
                keep = keep & (z >= down[:, s["top_k"] - 1:s["top_k"]])
            if s["top_p"] < 1:
                mass = torch.where(keep, w, 0.0).gather(1, order)
                upto = mass.cumsum(1)
                inside = upto - mass < s["top_p"] * upto[:, -1:]
                inside[:, 0] = True
                keep = keep & (z >= torch.where(inside, down, _INF).amin(1, keepdim=True))
        keep = keep & (w >= s["min_p"])
        key = torch.where(keep, z - torch.log(s["noise"]), -_INF)
    else:
        key = z
    best = key.amax(1, keepdim=True)
    index = torch.arange(v, device=x.device)
    token = torch.where(key == best, index, v).amin(1)
    logprob = z.gather(1, token[:, None]) - top - torch.log(total)
    none = best == -_INF
    return torch.where(none[:, 0], -1, token), torch.where(none, -_INF, logprob)[:, 0]


# ---------------------------------------------------------------------------- the floor
def work(c):
    if c["op"] == "int4":
        m, n, k = c["m"], c["n"], c["k"]
        e, groups = _SIZE[c["dtype"]], -(-c["k"] // c["group"])
        o = 4 if c["out"] == "f32" else e
        return {"bytes": n * k // 2 + groups * n * (e + (1 if c["zeros"] else 0)) + m * k * e + m * n * o
                + (n * e if c["bias"] else 0), "flops": 2 * m * n * k}
    b, v, e = c["b"], c["v"], _SIZE[c["dtype"]]
    if c["op"] == "process":
        o = 4 if c["out"] == "f32" else e
        # the mean row's list is filled to 0.65 of its length
        return {"bytes": b * v * (e + o) + int(0.65 * 8 * b * c["length"]) + 20 * b + 12 * b * c["biases"]
                + (b * v // 8 if c["mask"] else 0), "flops": 5 * b * v}
    kept = c["top_k"] if 0 < c["top_k"] < v else v
    noise = 0 if c["temperature"] == 0 else 4 * b * (kept if c["top_p"] == 1 and c["min_p"] == 0 else min(kept, 1000))
    return {"bytes": b * v * e + noise + 12 * b, "flops": 4 * b * v}


# ---------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"int4": _exact_int4, "process": _exact_process, "sample": _exact_sample}[case["op"]](s)


def _exact_int4(s):
    """Group by group: y += (x_g q_gᵀ - z sum x_g) s, each in 64 bits."""
    x, q, s_, z = s["x"].double(), s["q"], s["s"].double(), s["z"]
    m, k = x.shape
    n, group = q.shape[0], s["group"]
    y = torch.zeros(m, n, dtype=torch.float64, device=x.device)
    for j, lo in enumerate(range(0, k, group)):
        hi = min(lo + group, k)
        codes = q[:, lo // 2:hi // 2]
        part = x[:, lo:hi:2] @ (codes % 16).double().t() + x[:, lo + 1:hi:2] @ (codes // 16).double().t()
        shift = x[:, lo:hi].sum(1)[:, None] * (8.0 if z is None else z[j].double()[None])
        y += (part - shift) * s_[j][None]
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_process(s):
    host = {k: (t.double() if t.is_floating_point() else t).cpu().numpy() if isinstance(t, torch.Tensor) else t
            for k, t in s.items()}
    y = host["logits"].copy()
    b, v = y.shape
    for i in range(b):
        history, start = host["tokens"][i, :host["lengths"][i]], host["prompt"][i]
        made = np.bincount(history[start:], minlength=v)[:v].astype(np.float64)
        seen = np.unique(history)
        row = y[i]
        row[seen] = np.where(row[seen] > 0, row[seen] / host["r"][i], row[seen] * host["r"][i])
        row -= host["f"][i] * made
        row[made > 0] -= host["p"][i]
        if host["ids"] is not None:
            for t, value in zip(host["ids"][i], host["values"][i]):
                if 0 <= t < v:
                    row[t] += value
        if host["mask"] is not None:
            allowed = np.unpackbits(host["mask"][i].view(np.uint8), bitorder="little")[:v]
            row[allowed == 0] = -np.inf
    return torch.from_numpy(y)


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    noise = None if s["noise"] is None else s["noise"].double().cpu().numpy()
    b, v = logits.shape
    tokens, logprobs = np.full(b, -1, np.int64), np.full(b, -np.inf)
    for i in range(b):
        z = logits[i] / (s["t"] or 1.0)
        if not z.max() > -np.inf:
            continue
        weight = np.exp(z - z.max())
        if s["t"] == 0:
            tokens[i] = int(np.argmax(z))
        else:
            order = np.argsort(-z, kind="stable")
            kept = order[:v]
            if 0 < s["top_k"] < v:
                kept = order[z[order] >= z[order[s["top_k"] - 1]]]
            if s["top_p"] < 1:
                above = np.concatenate([[0.0], np.cumsum(weight[kept])])
                last = max(1, int(np.searchsorted(above[:-1], s["top_p"] * above[-1], side="left")))
                kept = kept[z[kept] >= z[kept[last - 1]]]
            kept = np.sort(kept[(weight[kept] >= s["min_p"]) & (z[kept] > -np.inf)])
            tokens[i] = kept[np.argmax(z[kept] - np.log(noise[i, kept]))]
        logprobs[i] = z[tokens[i]] - z.max() - math.log(weight.sum())
    return torch.from_numpy(tokens), torch.from_numpy(logprobs)
