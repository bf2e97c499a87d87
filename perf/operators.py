"""The state-space serving operators as one measures them: inputs, a plain form of each in elementary torch
operations, the package's calls, and the definitions in 64 bits.

Four operators make up a state-space layer served in 8 bits: rows quantised to int8 with a scale each
(``quantize``), the int8 product with scales for token and channel (``product``), the short causal
convolution (``conv``, ``conv_step``) and the selective scan (``scan``, ``scan_step``).  Sequences of a
prompt are packed along the token axis with offsets; states live in slots of a cache.
"""
import math
import os
import random
import sys

import torch

own = False  # True: run() makes the package's calls instead of the plain forms

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _package():
    if "kernelintrinsics" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "kernelintrinsics.jl_b200"))
    import kernelintrinsics

    return kernelintrinsics


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one long prompt through the convolution of a wide layer
        {"name": "conv prompt", "op": "conv", "type": "bf16", "tokens": 8192, "seqs": 1, "channels": 4096, "width": 4,
         "state": True, "carry": False, "silu": True},
        # a batch of ragged prompts, half of them continued from their slots, in Float32
        {"name": "conv ragged", "op": "conv", "type": "f32", "tokens": 5003, "seqs": 37, "channels": 1030, "width": 3,
         "state": True, "carry": True, "silu": True},
        # one decoding step of 64 requests
        {"name": "conv step", "op": "conv_step", "type": "bf16", "batch": 64, "channels": 4096, "width": 4, "silu": True},
        # the long prompt's scan, gated
        {"name": "scan prompt", "op": "scan", "type": "bf16", "tokens": 8192, "seqs": 1, "channels": 4096, "states": 16,
         "groups": 1, "gate": True, "softplus": True, "state": True, "carry": False},
        # ragged prompts of a smaller layer, two groups of B and C, half continued from their slots
        {"name": "scan ragged", "op": "scan", "type": "f32", "tokens": 6001, "seqs": 19, "channels": 1540, "states": 16,
         "groups": 2, "gate": False, "softplus": True, "state": True, "carry": True},
        # one decoding step of 128 requests
        {"name": "scan step", "op": "scan_step", "type": "bf16", "batch": 128, "channels": 4096, "states": 16, "groups": 1,
         "gate": True, "softplus": True},
        # a prompt's activations before a projection
        {"name": "quantize prompt", "op": "quantize", "type": "bf16", "rows": 8192, "cols": 4096},
        # a few tokens of a decoding step
        {"name": "quantize tokens", "op": "quantize", "type": "f16", "rows": 7, "cols": 8200},
        # a projection of one token: the weight's bytes are what counts
        {"name": "product token", "op": "product", "type": "bf16", "rows": 1, "channels": 4096, "inner": 4096, "bias": False},
        # a decoding step's projection of 48 tokens
        {"name": "product step", "op": "product", "type": "f16", "rows": 48, "channels": 8192, "inner": 4096, "bias": True},
        # sizes that fit no tile, rows that start at any byte
        {"name": "product ragged", "op": "product", "type": "f32", "rows": 1111, "channels": 4099, "inner": 2057, "bias": True},
        # a prompt's projection: the tensor cores' rate is what counts
        {"name": "product prompt", "op": "product", "type": "bf16", "rows": 8192, "channels": 8192, "inner": 4096, "bias": False},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm, odd ones among them."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _wide(rng, low, high, unit):
    """A width: mostly whole units as layers have them, now and then any number."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(unit, n // unit * unit)


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan", "scan_step", "quantize", "product", "product"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "conv":
        tokens = _spread(rng, 1, 16384)
        channels = _wide(rng, 64, 8192, 64)
        channels = max(64, min(channels, (8192 * 4096) // tokens))
        state = rng.random() < 0.7
        return {"op": op, "type": kind, "tokens": tokens, "seqs": _spread(rng, 1, 64), "channels": channels,
                "width": rng.choice([2, 3, 4, 4, 4]), "state": state, "carry": state and rng.random() < 0.5,
                "silu": rng.random() < 0.8}
    if op == "conv_step":
        return {"op": op, "type": kind, "batch": _spread(rng, 1, 512), "channels": _wide(rng, 64, 8192, 64),
                "width": rng.choice([2, 3, 4, 4, 4]), "silu": rng.random() < 0.8}
    if op == "scan":
        tokens = _spread(rng, 1, 8192)
        states = rng.choice([8, 16, 16, 16, 13, 32, 64])
        groups = rng.choice([1, 1, 1, 2])
        channels = _wide(rng, 64, 8192, 64)
        channels = max(64, min(channels, (8192 * 4096 * 16) // (tokens * states)))
        channels -= channels % groups
        state = rng.random() < 0.7
        return {"op": op, "type": kind, "tokens": tokens, "seqs": _spread(rng, 1, 32), "channels": channels,
                "states": states, "groups": groups, "gate": rng.random() < 0.6, "softplus": rng.random() < 0.8,
                "state": state, "carry": state and rng.random() < 0.5}
    if op == "scan_step":
        groups = rng.choice([1, 1, 1, 2])
        channels = _wide(rng, 64, 8192, 64)
        return {"op": op, "type": kind, "batch": _spread(rng, 1, 256), "channels": channels - channels % groups,
                "states": rng.choice([8, 16, 16, 13, 32]), "groups": groups, "gate": rng.random() < 0.6,
                "softplus": rng.random() < 0.8}
    if op == "quantize":
        rows = _spread(rng, 1, 16384)
        return {"op": op, "type": kind, "rows": rows, "cols": min(_wide(rng, 64, 16384, 64), (8192 * 8192) // rows)}
    rows = _spread(rng, 1, 8192)
    return {"op": op, "type": kind, "rows": rows, "channels": _wide(rng, 64, 8192, 64), "inner": _wide(rng, 64, 4096, 64),
            "bias": rng.random() < 0.4}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _offsets(seed, tokens, seqs):
    """Where each packed sequence starts: lengths of one token to long ones, an empty one now and then."""
    if seqs == 1:
        return [0, tokens]
    r = random.Random(seed * 7919 + 13)
    cuts = sorted(r.randint(0, tokens) for _ in range(seqs - 1))
    return [0] + cuts + [tokens]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype or t)

    def slots(n, more):
        return torch.randperm(n + more, generator=g, device=dev)[:n].to(torch.int32)

    s = dict(case)
    op = case["op"]
    if op in ("conv", "conv_step"):
        d, w = case["channels"], case["width"]
        s["weight"] = normal(d, w, scale=w ** -0.5)
        s["bias"] = normal(d, scale=0.1)
        n = case["seqs"] if op == "conv" else case["batch"]
        if op == "conv":
            # the convolution's input is one half of a projection's rows
            s["x"] = normal(case["tokens"], 2 * d)[:, :d]
            s["offsets"] = torch.tensor(_offsets(seed, case["tokens"], n), dtype=torch.int32, device=dev)
        else:
            s["x"] = normal(n, 2 * d)[:, :d]
        if op == "conv_step" or case["state"]:
            s["cache"] = normal(n + 3, w - 1, d)
            s["slots"] = slots(n, 3)
            s["initial"] = (torch.rand(n, generator=g, device=dev) < 0.5) if case.get("carry", True) else \
                torch.zeros(n, dtype=torch.bool, device=dev)
    elif op in ("scan", "scan_step"):
        d, k, gr = case["channels"], case["states"], case["groups"]
        n = case["seqs"] if op == "scan" else case["batch"]
        rows = case["tokens"] if op == "scan" else n
        s["u"] = torch.nn.functional.silu(normal(rows, d, dtype=torch.float32)).to(t)
        step = torch.exp(torch.rand(d, generator=g, device=dev) * math.log(100.0) + math.log(1e-3))  # 0.001 to 0.1
        if case["softplus"]:
            s["delta"] = normal(rows, d, scale=0.5)
            s["delta_bias"] = step + torch.log(-torch.expm1(-step))  # softplus's inverse
        else:
            s["delta"] = (step * torch.exp(normal(rows, d, scale=0.5, dtype=torch.float32))).to(t)
            s["delta_bias"] = None
        s["A"] = -torch.arange(1, k + 1, device=dev, dtype=torch.float32) * torch.exp(normal(d, k, scale=0.1, dtype=torch.float32))
        # B and C are slices of one projection's rows
        bc = normal(rows, 8 + 2 * gr * k)
        s["B"] = bc[:, 8:8 + gr * k].unflatten(1, (gr, k))
        s["C"] = bc[:, 8 + gr * k:].unflatten(1, (gr, k))
        s["D"] = 1 + normal(d, scale=0.1, dtype=torch.float32)
        s["z"] = normal(rows, 2 * d)[:, d:] if case["gate"] else None
        if op == "scan":
            s["offsets"] = torch.tensor(_offsets(seed, rows, n), dtype=torch.int32, device=dev)
        if op == "scan_step" or case["state"]:
            s["cache"] = normal(n + 3, d, k, scale=0.3, dtype=torch.float32)
            s["slots"] = slots(n, 3)
            s["initial"] = (torch.rand(n, generator=g, device=dev) < 0.5) if case.get("carry", True) else \
                torch.zeros(n, dtype=torch.bool, device=dev)
    elif op == "quantize":
        # activations: a few channels far larger than the others, rows of different sizes
        x = normal(case["rows"], case["cols"], dtype=torch.float32) * torch.exp(normal(case["rows"], 1, scale=0.5, dtype=torch.float32))
        loud = torch.rand(case["cols"], generator=g, device=dev) < 0.005
        s["x"] = torch.where(loud, x * 20, x).to(t)
    else:
        m, n, k = case["rows"], case["channels"], case["inner"]
        s["a"] = normal(m, k, scale=32, dtype=torch.float32).round().clamp(-127, 127).to(torch.int8)
        s["w"] = normal(n, k, scale=40, dtype=torch.float32).round().clamp(-127, 127).to(torch.int8)
        s["sa"] = torch.exp(normal(m, scale=0.5, dtype=torch.float32)) * 0.02
        s["sw"] = torch.exp(normal(n, scale=0.3, dtype=torch.float32)) * 0.0005
        s["bias"] = normal(n, scale=0.1, dtype=torch.float32) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
def _conv(s):
    x, w = s["x"], s["weight"]
    rows, d, width = x.shape[0], x.shape[1], w.shape[1]
    dev, taps = x.device, torch.arange(w.shape[1], device=x.device)
    cache = s.get("cache")
    start, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    seq = torch.searchsorted(s["offsets"][1:].long(), torch.arange(rows, device=dev), right=True)
    # the rows that are looked up: the tokens, then every sequence's initial inputs, then a row of zeros
    pool = [x.float()]
    if cache is not None:
        pool.append((cache[s["slots"].long()].float() * s["initial"][:, None, None]).reshape(-1, d))
    pool.append(torch.zeros(1, d, device=dev))
    pool = torch.cat(pool)

    def place(token, of):  # where token number `token` of sequence `of` lies in the pool
        before = rows + of * (width - 1) + (width - 1) + (token - start[of]) if cache is not None else \
            torch.full_like(token, rows)
        return torch.where(token >= start[of], token, before)

    near = place(torch.arange(rows, device=dev)[:, None] - (width - 1) + taps, seq[:, None].expand(rows, width))
    y = (pool[near] * w.float().t()).sum(1) + s["bias"].float()
    if s["silu"]:
        y = y * torch.sigmoid(y)
    if cache is not None:
        each = torch.arange(start.numel(), device=dev)[:, None].expand(-1, width - 1)
        last = place(end[:, None] - (width - 1) + taps[:-1], each)
        cache[s["slots"].long()] = pool[last].to(cache.dtype)
    return y.to(x.dtype), cache


def _conv_step(s):
    x, w, at = s["x"], s["weight"].float(), s["slots"].long()
    seen = torch.cat([s["cache"][at].float(), x.float()[:, None]], 1)  # batch, width, channels
    y = (seen * w.t()).sum(1) + s["bias"].float()
    if s["silu"]:
        y = y * torch.sigmoid(y)
    s["cache"][at] = seen[:, 1:].to(s["cache"].dtype)
    return y.to(x.dtype), s["cache"]


def _steps(s):
    """Per token and channel: the step, and per state: the decay and what is added."""
    dt = s["delta"].float()
    if s["delta_bias"] is not None:
        dt = dt + s["delta_bias"]
    if s["softplus"]:
        dt = torch.where(dt > 20, dt, torch.log1p(torch.exp(dt.clamp(max=20))))
    per = s["u"].shape[1] // s["groups"]
    b, c = (s[k].float().repeat_interleave(per, 1) for k in ("B", "C"))  # rows, channels, states
    decay = torch.exp(dt[:, :, None] * s["A"])
    return decay, (dt * s["u"].float())[:, :, None] * b, c


def _out(s, h, c):
    y = (h * c).sum(2) + s["D"] * s["u"].float()
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    return y.to(s["u"].dtype)


def _scan(s):
    decay, h, c = _steps(s)
    cache, rows = s.get("cache"), h.shape[0]
    start, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    full = end > start
    first = start[full]
    if cache is not None:
        at = s["slots"].long()
        before = cache[at] * s["initial"][:, None, None]
        h[first] += decay[first] * before[full]
    decay[first] = 0  # no sequence sees the one before it
    reach = 1
    while reach < rows:  # every token takes in twice as many tokens before it each time
        h = torch.cat([h[:reach], h[reach:] + decay[reach:] * h[:-reach]])
        decay = torch.cat([decay[:reach], decay[reach:] * decay[:-reach]])
        reach *= 2
    if cache is not None:
        cache[at] = torch.where(full[:, None, None], h[(end - 1).clamp(min=0)], before)
    return _out(s, h, c), cache


def _scan_step(s):
    decay, add, c = _steps(s)
    at = s["slots"].long()
    h = s["cache"][at] * decay + add
    s["cache"][at] = h
    return _out(s, h, c), s["cache"]


def _quantize(s):
    x = s["x"].float()
    scale = x.abs().amax(1) / 127.0
    q = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0)
    return q.round().clamp(-127, 127).to(torch.int8), scale  # the int8 are whole numbers


def _product(s):
    y = (s["a"].float() @ s["w"].float().t()) * s["sa"][:, None] * s["sw"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(_TYPES[s["type"]])


_PLAIN = {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "quantize": _quantize,
          "product": _product}


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return _PLAIN[s["op"]](s)
    KI = _package()
    act = "silu" if s.get("silu") else None
    if s["op"] == "conv":
        y = KI.causal_conv(s["x"], s["weight"], s["bias"], state=s.get("cache"), offsets=s["offsets"], slots=s.get("slots"),
                           initial=s.get("initial"), activation=act)
        return y, s.get("cache")
    if s["op"] == "conv_step":
        return KI.causal_conv_step(s["x"], s["weight"], s["bias"], state=s["cache"], slots=s["slots"], activation=act), s["cache"]
    if s["op"] == "scan":
        y = KI.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                              softplus=s["softplus"], state=s.get("cache"), offsets=s["offsets"], slots=s.get("slots"),
                              initial=s.get("initial"))
        return y, s.get("cache")
    if s["op"] == "scan_step":
        y = KI.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                   delta_bias=s["delta_bias"], softplus=s["softplus"], state=s["cache"], slots=s["slots"])
        return y, s["cache"]
    if s["op"] == "quantize":
        return KI.quantize_rows(s["x"])
    return KI.int8_gemm(s["a"], s["w"], s["sa"], s["sw"], bias=s["bias"], dtype=_TYPES[s["type"]])


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _runs(s):
    """(first row, row behind the last) of each sequence, in order."""
    o = s["offsets"].tolist() if "offsets" in s else list(range(s["batch"] + 1))
    return list(zip(o[:-1], o[1:]))


def exact(case, seed):
    s = prepare(case, seed)
    op, f = case["op"], torch.float64
    if op == "quantize":
        return None, s["x"].to(f).abs().max(dim=1).values / 127
    if op == "product":
        y = torch.mm(s["a"].to(f), s["w"].to(f).T) * torch.outer(s["sa"].to(f), s["sw"].to(f))
        return y if s["bias"] is None else y + s["bias"].to(f)
    cache = s["cache"].to(f) if "cache" in s else None
    at = s["slots"].tolist() if cache is not None else None
    keep = s["initial"].tolist() if cache is not None and "offsets" in s else None
    if op in ("conv", "conv_step"):
        w, x = s["weight"].to(f), s["x"].to(f)
        d, width = w.shape
        y = torch.zeros_like(x)
        for i, (lo, hi) in enumerate(_runs(s)):
            head = torch.zeros(width - 1, d, dtype=f, device=x.device)
            if cache is not None and (keep is None or keep[i]):
                head = cache[at[i]].clone()
            line = torch.cat([head, x[lo:hi]])
            for j in range(width):
                y[lo:hi] += line[j:j + hi - lo] * w[:, j]
            if cache is not None:
                cache[at[i]] = line[hi - lo:]
        y += s["bias"].to(f)
        return (y / (1 + torch.exp(-y)) if s["silu"] else y), cache
    dt = s["delta"].to(f) + (0 if s["delta_bias"] is None else s["delta_bias"].to(f))
    if s["softplus"]:
        dt = torch.logaddexp(dt, torch.zeros_like(dt))
    u, A, spans = s["u"].to(f), s["A"].to(f), _runs(s)
    per = u.shape[1] // case["groups"]
    h = torch.zeros(len(spans), *A.shape, dtype=f, device=u.device)
    if cache is not None:
        for i in range(len(spans)):
            if keep is None or keep[i]:
                h[i] = cache[at[i]]
    y = torch.zeros_like(u)
    lengths = [hi - lo for lo, hi in spans]
    order = sorted(range(len(spans)), key=lambda i: -lengths[i])  # the longest first: the live ones are a prefix
    h = h[order]
    firsts = torch.tensor([spans[i][0] for i in order], device=u.device)
    live = len(order)
    for t in range(max(lengths)):
        while lengths[order[live - 1]] <= t:
            live -= 1
        row = firsts[:live] + t
        b, c = (s[k][row].to(f).repeat_interleave(per, dim=1) for k in ("B", "C"))
        d_t = dt[row].unsqueeze(-1)
        h[:live] = torch.exp(d_t * A) * h[:live] + d_t * u[row].unsqueeze(-1) * b
        y[row] = (h[:live] * c).sum(-1)
    y += s["D"].to(f) * u
    if s["z"] is not None:
        z = s["z"].to(f)
        y *= z / (1 + torch.exp(-z))
    if cache is not None:
        for i, q in enumerate(order):
            cache[at[q]] = h[i]
    return y, cache


# ---------------------------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    op, e = case["op"], _SIZE[case["type"]]
    if op in ("conv", "conv_step"):
        d, w = case["channels"], case["width"]
        rows, n = (case["tokens"], case["seqs"]) if op == "conv" else (case["batch"], case["batch"])
        held = n * (w - 1) * d * e if op == "conv_step" or case["state"] else 0
        read = held if op == "conv_step" or case.get("carry") else 0
        return {"bytes": 2 * rows * d * e + d * (w + 1) * e + held + read, "flops": rows * d * (2 * w + (4 if case["silu"] else 0))}
    if op in ("scan", "scan_step"):
        d, k, g = case["channels"], case["states"], case["groups"]
        rows, n = (case["tokens"], case["seqs"]) if op == "scan" else (case["batch"], case["batch"])
        held = n * d * k * 4 if op == "scan_step" or case["state"] else 0
        read = held if op == "scan_step" or case.get("carry") else 0
        # the product with A, the exponential, what is added, the recurrence (2), the sum over C (2)
        return {"bytes": rows * d * e * (4 if case["gate"] else 3) + rows * 2 * g * k * e + d * (k + 2) * 4 + held + read,
                "flops": rows * d * (7 * k + 8)}
    if op == "quantize":
        return {"bytes": case["rows"] * case["cols"] * (e + 1) + 4 * case["rows"], "flops": 3 * case["rows"] * case["cols"]}
    m, n, k = case["rows"], case["channels"], case["inner"]
    return {"bytes": m * k + n * k + m * n * e + 4 * (m + n), "flops": 2 * m * n * k}
