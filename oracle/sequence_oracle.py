"""numpy restatement, in float64, of the sequence operators (``sequence.py``), each with a bound on what an evaluation in
another precision may be off.

The bounds are running error analyses: every elementary step may be off by ``k`` units (``u``, half a step of the
arithmetic's type at 1) relative to the magnitudes it adds, and errors pass through the formulas by the triangle
inequality.  ``k`` covers the exponential, the quotient and the few roundings of one step (``STEP``); a sum of ``m`` terms
may be off by ``m`` units of the sum of their magnitudes, whatever the order.  The caller adds the final rounding to the
output's type.
"""
import math

import numpy as np

STEP = 16.0  # units a step may be off: exp 2 + |argument| <= 8, quotient 2, products and sums 4


def gate_step(g):
    """Units that a step with the sigmoid of ``g`` may be off: the exponential's argument g log2(e) is rounded, and log2(e)
    itself, which makes 1.22 |g| of them beyond what the eight in STEP cover."""
    g = np.abs(g)
    return np.where(g <= 8, STEP, 8 + 1.25 * g)


def sigmoid(g):
    with np.errstate(over="ignore"):
        return np.where(g >= 0, 1 / (1 + np.exp(-np.abs(g))), np.exp(-np.abs(g)) / (1 + np.exp(-np.abs(g))))


def recurrence(x, gate, initial=None, lens=None, reverse=False, grad_y=None, grad_final=None, u=2.0 ** -24):
    """Values and bounds: dict of name -> (value, bound).  Frames behind an utterance's end are not looked at."""
    n, t, c = x.shape
    lens = np.full(n, t) if lens is None else np.clip(np.asarray(lens), 0, t)
    out = {name: (np.zeros((n, t, c)), np.zeros((n, t, c))) for name in ("y", "grad_x", "grad_gate")}
    final = (np.zeros((n, c)), np.zeros((n, c)))
    first = (np.zeros((n, c)), np.zeros((n, c)))
    for i in range(n):
        order = range(int(lens[i]))
        order = list(reversed(order)) if reverse else list(order)
        h = np.zeros(c) if initial is None else initial[i].astype(np.float64)
        e = np.zeros(c)
        before = {}
        for j in order:
            f, keep, k = sigmoid(gate[i, j]), sigmoid(-gate[i, j]), gate_step(gate[i, j]) * u
            before[j] = (h, e)
            e = f * e + k * (f * np.abs(h) + keep * np.abs(x[i, j]))
            h = f * h + keep * x[i, j]
            out["y"][0][i, j], out["y"][1][i, j] = h, e
        final[0][i], final[1][i] = h, e
        m = np.zeros(c) if grad_final is None else grad_final[i].astype(np.float64)
        e = np.zeros(c)
        for j in reversed(order):
            f, keep, k = sigmoid(gate[i, j]), sigmoid(-gate[i, j]), gate_step(gate[i, j]) * u
            gy = np.zeros(c) if grad_y is None else grad_y[i, j]
            gh, eh = gy + m, e + k * (np.abs(gy) + np.abs(m))
            hb, eb = before[j]
            d, ed = hb - x[i, j], eb + k * (np.abs(hb) + np.abs(x[i, j]))
            out["grad_x"][0][i, j], out["grad_x"][1][i, j] = keep * gh, keep * (eh + k * np.abs(gh))
            out["grad_gate"][0][i, j] = f * keep * gh * d
            out["grad_gate"][1][i, j] = f * keep * (eh * np.abs(d) + np.abs(gh) * ed + k * np.abs(gh * d) + eh * ed)
            m, e = f * gh, f * (eh + k * np.abs(gh))
        first[0][i], first[1][i] = m, e
    out["final"], out["grad_initial"] = final, first
    return out


def _erf(z):
    return np.vectorize(math.erf)(z) if z.size else z


def activation(z, act):
    """Value, slope and a bound on the slope's own slope."""
    if act == "none":
        return z, np.ones_like(z), 0.0
    if act == "relu":
        return np.maximum(z, 0), (z > 0).astype(np.float64), 0.0
    if act == "silu":
        s = sigmoid(z)
        return z * s, s * (1 + z * sigmoid(-z)), 0.5
    cdf = 0.5 * (1 + _erf(z / math.sqrt(2)))
    return z * cdf, cdf + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8


def group_norm_act(x, groups, weight=None, bias=None, lens=None, eps=1e-5, act="none", grad_y=None, u=2.0 ** -24):
    """Values and bounds on a (batch, frames, channels) input."""
    n, t, c = x.shape
    lens = np.full(n, t) if lens is None else np.clip(np.asarray(lens), 0, t)
    w = np.ones(c) if weight is None else weight.astype(np.float64)
    b = np.zeros(c) if bias is None else bias.astype(np.float64)
    y, gx = (np.zeros((n, t, c)), np.zeros((n, t, c))), (np.zeros((n, t, c)), np.zeros((n, t, c)))
    gw, gb, sw, sb = (np.zeros(c), np.zeros(c)), (np.zeros(c), np.zeros(c)), np.zeros(c), np.zeros(c)
    k = STEP * u
    for i in range(n):
        length = int(lens[i])
        if length == 0:
            continue
        ks = (64 + length) * u  # a thread adds at most a group's frames one after the other, the rest is a short tree

        def mean(v):
            return np.broadcast_to(v.reshape(length, groups, -1).mean((0, 2))[None, :, None],
                                   (length, groups, c // groups)).reshape(length, c)

        v = x[i, :length].astype(np.float64)
        d = v - mean(v)
        e_d = ks * mean(np.abs(v)) + k * (np.abs(v) + np.abs(mean(v)))
        var = mean(d * d)
        e_var = mean(2 * np.abs(d) * e_d + e_d * e_d) + ks * var
        rstd = 1 / np.sqrt(var + eps)
        e_rstd = rstd * (0.5 * e_var * rstd * rstd + k)
        xhat = d * rstd
        e_xhat = e_d * rstd + np.abs(d) * e_rstd + e_d * e_rstd + k * np.abs(xhat)
        z = xhat * w + b
        e_z = np.abs(w) * e_xhat + k * (np.abs(xhat * w) + np.abs(b))
        a, slope, bend = activation(z, act)
        y[0][i, :length], y[1][i, :length] = a, 1.13 * e_z + k * np.abs(z)
        if grad_y is None:
            continue
        gy = grad_y[i, :length].astype(np.float64)
        gz = gy * slope
        e_gz = np.abs(gy) * (bend * e_z + k * (1 + np.abs(z) * (act in ("silu", "gelu"))))
        if act == "relu":  # either side of the corner is right where z may be off across it
            e_gz = e_gz + np.abs(gy) * (np.abs(z) <= e_z)
        q, e_q = gz * w, np.abs(w) * e_gz + k * np.abs(gz * w)
        s1, e_s1 = mean(q), mean(e_q) + ks * mean(np.abs(q))
        s2 = mean(q * xhat)
        e_s2 = mean(e_q * np.abs(xhat) + np.abs(q) * e_xhat + e_q * e_xhat) + ks * mean(np.abs(q * xhat))
        gx[0][i, :length] = rstd * (q - s1 - xhat * s2)
        size = np.abs(q) + np.abs(s1) + np.abs(xhat * s2)
        gx[1][i, :length] = (rstd * (e_q + e_s1 + np.abs(xhat) * e_s2 + e_xhat * np.abs(s2) + e_xhat * e_s2 + k * size)
                             + e_rstd * size)
        gw[0][:] += (gz * xhat).sum(0)
        gw[1][:] += (e_gz * np.abs(xhat) + np.abs(gz) * e_xhat + e_gz * e_xhat).sum(0)
        sw += np.abs(gz * xhat).sum(0) * (64 + length + n)
        gb[0][:] += gz.sum(0)
        gb[1][:] += e_gz.sum(0)
        sb += np.abs(gz).sum(0) * (64 + length + n)
    gw[1][:] += sw * u
    gb[1][:] += sb * u
    return {"y": y, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}


def philox4x32_10(counters, key):
    """(count, 4) words of Philox4x32-10 for 64-bit counters (the upper two counter words zero) and a 64-bit key."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    counters = np.asarray(counters, dtype=np.uint64)
    c = [counters & low, counters >> half, np.zeros_like(counters), np.zeros_like(counters)]
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & low, (a >> half) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1)


def dropout_keep(shape, p, seed):
    """Truth values: which elements are kept."""
    count = int(np.prod(shape, dtype=np.int64))
    words = philox4x32_10(np.arange((count + 3) // 4), seed).reshape(-1)[:count]
    return (words >= np.uint64(int(math.floor(p * 2.0 ** 32 + 0.5)))).reshape(shape)
