"""Plain 64-bit forms of the layer operators (numpy), with bounds on what Float32 arithmetic may be off.

A bound follows the formula: every Float32 operation is off by at most half a step (2^-24 relative), the fast
exponential by 2 ulp (2^-22) plus the rounding of its argument, a division by 2 ulp; a stored result by half a
step of its type.  Sums of products are bounded by their absolute values.
"""
from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -24  # half a step of Float32
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-36, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-36}  # half a subnormal step, flushed tails


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def silu(s, err):
    """(silu(s), bound): the exponential's relative error is (4 + 3|s|) 2^-24 * 2, two more operations and a
    division (2 ulp) follow; |silu'| <= 1.1 passes the argument's error on."""
    y = s / (1 + np.exp(-s))
    return y, 1.1 * err + (16 + 6 * np.abs(s)) * U * np.abs(y)


def stored(y, err, dtype):
    """The bound of a result after it is rounded to dtype."""
    return err + HALF_STEP[dtype] * (np.abs(y) + err) + TINY[dtype]


def conv(x, w, bias, spans, states, act):
    """y, bound and final states; x: tokens x channels, w: channels x width, spans: (begin, end) per sequence, states:
    (width-1) x channels arrays of the state each sequence starts from."""
    width = w.shape[1]
    y, err = np.zeros_like(x), np.zeros_like(x)
    last = []
    for (b, e), st in zip(spans, states):
        line = np.concatenate([st, x[b:e]])
        s = np.zeros((e - b, x.shape[1])) + (0 if bias is None else bias)
        mag = np.abs(s)
        for j in range(width):
            s += line[j:j + e - b] * w[:, j]
            mag += np.abs(line[j:j + e - b] * w[:, j])
        er = (width + 1) * U * mag
        if act:
            s, er = silu(s, er)
        y[b:e], err[b:e] = s, er
        last.append(line[e - b:])
    return y, err, last


def scan(u, delta, A, B, C, D, z, delta_bias, soft, spans, states):
    """y, its bound, final states and their bounds; B, C: tokens x groups x states."""
    channels, n = A.shape
    per = channels // B.shape[1]
    y, yerr = np.zeros_like(u), np.zeros_like(u)
    last, lasterr = [], []
    for (b, e), st in zip(spans, states):
        h, mag, err = st.copy(), np.abs(st), np.zeros_like(st)
        for t in range(b, e):
            x = delta[t] + (0 if delta_bias is None else delta_bias)
            xerr = U * np.abs(x)
            if soft:
                s = np.logaddexp(x, 0)
                # log1p and exp to 2 ulp each; relative error of softplus per error of x is at most 1
                rel = 8 * U + xerr + np.where(x > 20, 3e-9, 0)
            else:
                s, rel = x, U * np.ones_like(x)
            s, rel = s[:, None], rel[:, None]
            bt, ct = np.repeat(B[t], per, 0), np.repeat(C[t], per, 0)
            a = np.exp(s * A)
            add = s * u[t][:, None] * bt
            arel = 4 * U + 3 * U * np.abs(s * A) * 1.4427 + np.abs(s * A) * rel
            err = a * (1 + arel) * err + arel * a * mag + (rel + 4 * U) * np.abs(add) + 2.0 ** -126
            h = a * h + add
            mag = a * mag + np.abs(add)
            err = err + 2 * U * mag
            o = (ct * h).sum(1)
            oerr = (np.abs(ct) * err).sum(1) + (n + 4) * U * (np.abs(ct) * mag).sum(1)
            if D is not None:
                o = o + D * u[t]
                oerr = oerr + 2 * U * np.abs(D * u[t]) + U * np.abs(o)
            if z is not None:
                gate, gerr = silu(z[t], 0.0)
                oerr = oerr * (np.abs(gate) + gerr) + np.abs(o) * gerr + 2 * U * np.abs(o * gate)
                o = o * gate
            y[t], yerr[t] = o, oerr
        last.append(h)
        lasterr.append(err)
    return y, yerr, last, lasterr


def quantize(x):
    """scale and int8 of Float32 rows, by IEEE Float32 operations as the operator is defined (bit for bit)."""
    x = x.astype(np.float32)
    bits = np.abs(x).view(np.uint32)
    top = bits.max(1).view(np.float32) if x.shape[1] else np.zeros(x.shape[0], np.float32)
    with np.errstate(all="ignore"):
        scale = (top * (np.float32(1) / np.float32(127))).astype(np.float32)
        q = np.rint((x / scale[:, None]).astype(np.float32))
        q = np.where(np.isnan(q) | (scale[:, None] == 0), 0, np.clip(q, -127, 127))
    return scale, q.astype(np.int8)


def product(a, w, sa, sw, bias):
    """The product and its bound: an exact integer sum, rounded to Float32, two scalings and one addition."""
    s = (a.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64) * sa[:, None] * sw
    err = 4 * U * np.abs(s)
    if bias is not None:
        s = s + bias
        err = err + U * np.abs(s)
    return s, err
