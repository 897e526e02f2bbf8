"""The sequence operators on the calls that a user of the acoustic models makes: what is timed, and what it is held to.

Three operators that belong together, on per-frame features (batch, frames, channels), channels last:

* ``recurrence``: ``h_t = f_t h_{t-1} + (1 - f_t) x_t`` with ``f = sigmoid(gate)``, over ragged utterances, either way;
* ``norm``: group norm over an utterance's frames, then an activation;
* ``dropout``: a mask from the counter-based generator Philox4x32-10, never stored, optionally added to a residual.

A training case is one forward and one backward call and returns the output and every gradient.  With ``own`` false the
operators are written out in elementary torch operations in 32 bits, rounded once at the end; with ``own`` true they are
the calls of ``sequence.py``.  ``exact`` computes the same from the definitions in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cnn-mellin_b200")
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPS = 1e-5


def _sequence():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import sequence

    return sequence


# ---- the cases ---------------------------------------------------------------------------------------------------


def _recurrence(name, n, t, c, dtype, train, packed=True, ragged=True, shortest=0, initial=False, reverse=False):
    return {"name": name, "op": "recurrence", "n": n, "t": t, "c": c, "dtype": dtype, "train": train, "packed": packed,
            "ragged": ragged, "shortest": shortest, "initial": initial, "reverse": reverse}


def _norm(name, n, t, c, groups, dtype, train, act, ragged=True, shortest=0):
    return {"name": name, "op": "norm", "n": n, "t": t, "c": c, "groups": groups, "dtype": dtype, "train": train,
            "act": act, "ragged": ragged, "shortest": shortest}


def _dropout(name, n, t, c, p, dtype, train, residual):
    return {"name": name, "op": "dropout", "n": n, "t": t, "c": c, "p": p, "dtype": dtype, "train": train,
            "residual": residual}


def listed():
    return [
        # one frame of 64 streams at the model's hidden width, the state carried from call to call
        _recurrence("recurrence one frame bf16", 64, 1, 1024, "bfloat16", False, ragged=False, initial=True),
        # decoding a batch of utterances of 200 to 800 frames
        _recurrence("recurrence decode bf16", 32, 800, 1024, "bfloat16", False, shortest=200),
        # the training step's batch and precision
        _recurrence("recurrence train f32", 32, 800, 1024, "float32", True, shortest=200),
        # long recordings, few channels: the time axis is all the parallelism there is
        _recurrence("recurrence train long bf16", 2, 16384, 256, "bfloat16", True, ragged=False, initial=True),
        # the backward direction of a two-way layer, odd sizes, one utterance without a frame, separate tensors
        _recurrence("recurrence train odd f16", 5, 803, 333, "float16", True, packed=False, reverse=True),
        # a chunk of one stream
        _norm("norm one chunk f32", 1, 41, 256, 8, "float32", False, "relu", ragged=False),
        # the training step's batch and precision
        _norm("norm train f32", 32, 800, 1024, 32, "float32", True, "relu", shortest=200),
        # long recordings: a group of one utterance does not fit a multiprocessor
        _norm("norm train long bf16", 4, 16384, 256, 8, "bfloat16", True, "silu", ragged=False),
        # odd sizes, groups of 30 channels, one utterance without a frame
        _norm("norm train odd f16", 7, 411, 330, 11, "float16", True, "gelu"),
        # one frame of 64 streams
        _dropout("dropout one frame bf16", 64, 1, 1024, 0.05, "bfloat16", False, False),
        # the training step's batch and precision
        _dropout("dropout train f32", 32, 800, 1024, 0.05, "float32", True, False),
        # the end of a residual block, odd sizes
        _dropout("dropout train residual bf16", 31, 797, 1021, 0.2, "bfloat16", True, True),
    ]


_MOST = 32 * 800 * 1024


def _between(rng, lo, hi):
    """Spread over the logarithm; every second value odd, the other often a multiple of a power of two."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))
    v = min(max(v, lo), hi)
    if rng.random() < 0.5:
        return v | 1 if (v | 1) <= hi else v
    step = 1 << max(0, v.bit_length() - 3)
    return max(lo, v // step * step)


def draw(rng):
    op = rng.choice(["recurrence", "norm", "dropout"])
    n, t, c = _between(rng, 1, 64), _between(rng, 1, 16384), _between(rng, 8, 2048)
    while n * t * c > _MOST:
        if n > 1 and rng.random() < 0.5:
            n = (n + 1) // 2
        elif t >= c:
            t = (t + 1) // 2
        else:
            c = (c + 1) // 2
    dtype, train = rng.choice(["float32", "bfloat16", "float16"]), rng.random() < 0.7
    ragged = rng.random() < 0.6
    shortest = rng.choice([0, t // 4])
    if op == "recurrence":
        case = _recurrence("", n, t, c, dtype, train, rng.random() < 0.6, ragged, shortest, rng.random() < 0.5,
                           rng.random() < 0.4)
    elif op == "norm":
        groups = rng.choice([g for g in (1, 2, 3, 4, 8, 16, 32) if g <= c])
        case = _norm("", n, t, max(groups, c // groups * groups), groups, dtype, train,
                     rng.choice(["none", "relu", "silu", "gelu"]), ragged, shortest)
    else:
        case = _dropout("", n, t, c, rng.choice([0.05, 0.1, 0.2, 0.5]), dtype, train, rng.random() < 0.5)
    del case["name"]
    return case


def _lengths(case):
    """Frames of each utterance: spread from the shortest to t, dealt out in an order that is not sorted."""
    n, t = case["n"], case["t"]
    if not case.get("ragged"):
        return [t] * n
    lo = min(case["shortest"], t)
    order = sorted(range(n), key=lambda i: (i * 7919 + 13) % 104729)
    return [lo + (t - lo) * order[i] // max(n - 1, 1) if n > 1 else t for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, n, t, c = _DTYPES[case["dtype"]], case["n"], case["t"], case["c"]
    train = case["train"]

    def normal(*shape, mean=0.0, std=1.0, like=dtype, leaf=train):
        v = torch.randn(*shape, device="cuda", generator=gen).mul_(std).add_(mean).to(like)
        return v.requires_grad_(True) if leaf else v

    state = {"case": dict(case)}
    if case["op"] == "recurrence":
        # gates as a trained layer has them: mostly remembering
        if case["packed"]:
            mix = torch.randn(n, t, 2 * c, device="cuda", generator=gen)
            mix[..., c:] += 1.0
            state["x"], state["gate"] = mix.to(dtype).requires_grad_(train), None
        else:
            state["x"], state["gate"] = normal(n, t, c), normal(n, t, c, mean=1.0)
        state["initial"] = normal(n, c, like=torch.float32) if case["initial"] else None
        state["grad_y"] = normal(n, t, c, leaf=False) if train else None
        state["grad_final"] = normal(n, c, like=torch.float32, leaf=False) if train else None
    elif case["op"] == "norm":
        state["x"] = normal(n, t, c, mean=0.5, std=1.5)
        state["weight"] = normal(c, mean=1.0, std=0.2, like=torch.float32)
        state["bias"] = normal(c, std=0.2, like=torch.float32)
        state["grad_y"] = normal(n, t, c, leaf=False) if train else None
    else:
        state["x"] = normal(n, t, c)
        state["residual"] = normal(n, t, c) if case["residual"] else None
        state["grad_y"] = normal(n, t, c, leaf=False) if train else None
        state["seed"] = (int(seed) * 2654435761 + 12345) & ((1 << 62) - 1)
    if case["op"] != "dropout":
        state["lens"] = (torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None)
    return state


def work(case):
    """A training pass is two calls with the rest of the model between them: each reads its inputs and writes its
    outputs once.  Frames behind an utterance's end are never read; their outputs are written as zeros."""
    size = 4 if case["dtype"] == "float32" else 2
    n, t, c = case["n"], case["t"], case["c"]
    every, live = n * t * c, sum(_lengths(case)) * c
    if case["op"] == "recurrence":
        total = (2 * live + every) * size + 4 * n * c * (2 if case["initial"] else 1)
        flops = 8 * live
        if case["train"]:
            total += (3 * live + 2 * every) * size + 4 * n * c * (3 if case["initial"] else 1)
            flops += 16 * live
    elif case["op"] == "norm":
        total = (live + every) * size + 8 * c
        flops = 8 * live
        if case["train"]:
            total += (2 * live + every) * size + 16 * c
            flops += 20 * live
    else:
        total = (3 if case["residual"] else 2) * every * size
        flops = 2 * every
        if case["train"]:  # the residual's gradient is the output's
            total += 2 * every * size
            flops += 2 * every
    return {"bytes": total, "flops": flops}


# ---- the framework's calls ---------------------------------------------------------------------------------------


def _run_own(s):
    sequence, case = _sequence(), s["case"]
    if case["op"] == "recurrence":
        y, final = sequence.gated_recurrence(s["x"], s["gate"], s["initial"], s["lens"], case["reverse"])
        out = {"y": y, "final": final}
        if case["train"]:
            names = ["x"] + (["gate"] if s["gate"] is not None else []) + (["initial"] if s["initial"] is not None else [])
            grads = torch.autograd.grad([y, final], [s[k] for k in names], [s["grad_y"], s["grad_final"]])
            out.update({"grad_" + k: g for k, g in zip(names, grads)})
    elif case["op"] == "norm":
        y = sequence.group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], s["lens"], _EPS, case["act"])
        out = {"y": y}
        if case["train"]:
            grads = torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["grad_y"])
            out.update(zip(("grad_x", "grad_weight", "grad_bias"), grads))
    else:
        y = sequence.philox_dropout(s["x"], case["p"], True, s["seed"], s["residual"])
        out = {"y": y}
        if case["train"]:
            names = ["x"] + (["residual"] if s["residual"] is not None else [])
            grads = torch.autograd.grad(y, [s[k] for k in names], s["grad_y"])
            out.update({"grad_" + k: g for k, g in zip(names, grads)})
    return out


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _scan(a, b):
    """``h_t = a_t h_{t-1} + b_t`` along dim 1 from ``h_{-1} = 0``, by doubling: log2(t) passes."""
    step, t = 1, a.shape[1]
    while step < t:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def _live(case, lens):
    """(n, t, 1) truth values: frames inside their utterance; None where all are."""
    if lens is None:
        return None
    return (torch.arange(case["t"], device="cuda")[None, :] < lens[:, None])[..., None]


def _turned(v, lens, reverse):
    """The frames in the order in which the recurrence meets them (its own inverse)."""
    if not reverse:
        return v
    n, t, _ = v.shape
    at = torch.arange(t, device=v.device)[None, :].expand(n, t)
    length = (lens if lens is not None else torch.full((n,), t, device=v.device)).long()[:, None]
    at = torch.where(at < length, length - 1 - at, at)
    return torch.gather(v, 1, at[..., None].expand_as(v))


def _plain_recurrence(s):
    case, lens, c = s["case"], s["lens"], s["case"]["c"]
    dtype, live, rev = s["x"].dtype, _live(case, lens), case["reverse"]
    x, gate = (s["x"][..., :c], s["x"][..., c:]) if s["gate"] is None else (s["x"], s["gate"])
    x, gate = _turned(x.detach().float(), lens, rev), _turned(gate.detach().float(), lens, rev)
    f, keep = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    u = keep * x
    if live is not None:  # behind the end the state stays as it is
        f, u = torch.where(live, f, 1.0), torch.where(live, u, 0.0)
    h0 = s["initial"].detach() if s["initial"] is not None else torch.zeros(case["n"], c, device="cuda")
    u = torch.cat((u[:, :1] + f[:, :1] * h0[:, None], u[:, 1:]), 1)
    h = _scan(f, u)
    y = _turned(h if live is None else torch.where(live, h, 0.0), lens, rev).to(dtype)
    out = {"y": y, "final": h[:, -1].clone()}
    if not case["train"]:
        return out
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    gy = _turned(s["grad_y"].float(), lens, rev)
    if live is not None:
        gy = torch.where(live, gy, 0.0)
    # message from the frames after t: m_{t-1} = f_t (gy_t + m_t); gh_t = gy_t + m_t
    gy = torch.cat((gy[:, :-1], gy[:, -1:] + s["grad_final"][:, None]), 1)
    later = torch.cat((torch.ones_like(f[:, :1]), f[:, 1:].flip(1)), 1)
    gh = _scan(later, gy.flip(1)).flip(1)
    gx, gg = keep * gh, gh * (before - x) * f * keep
    if live is not None:
        gx, gg = torch.where(live, gx, 0.0), torch.where(live, gg, 0.0)
    gx, gg = _turned(gx, lens, rev).to(dtype), _turned(gg, lens, rev).to(dtype)
    if s["gate"] is None:
        out["grad_x"] = torch.cat((gx, gg), 2)
    else:
        out["grad_x"], out["grad_gate"] = gx, gg
    if s["initial"] is not None:
        out["grad_initial"] = f[:, 0] * gh[:, 0]
    return out


def _erf(z):
    """erf by the Maclaurin series where it is short, else 1 - erfc by Laplace's continued fraction, in 64 bits."""
    z = z.double()
    a = z.abs()
    small, term, total = a.clamp(max=3.0), None, None
    term = small.clone()
    total = small.clone()
    for k in range(1, 60):
        term = term * (-small * small / k)
        total = total + term / (2 * k + 1)
    big, frac = a.clamp(min=3.0), torch.zeros_like(a)
    for k in range(40, 0, -1):
        frac = (k / 2) / (big + frac)
    tail = 1 - torch.exp(-big * big) / ((big + frac) * math.sqrt(math.pi))
    return torch.sign(z) * torch.where(a < 3.0, total * (2 / math.sqrt(math.pi)), tail)


def _act(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return z * sig, sig * (1 + z * (1 - sig))
    phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    cdf = (0.5 * (1 + torch.erf(z / math.sqrt(2))))
    return z * cdf, cdf + z * phi


def _plain_norm(s):
    case, lens, groups = s["case"], s["lens"], s["case"]["groups"]
    n, t, c = case["n"], case["t"], case["c"]
    live, x = _live(case, lens), s["x"].detach().float()
    if live is not None:
        x = torch.where(live, x, 0.0)
    count = (lens.float() if lens is not None else torch.full((n,), float(t), device="cuda")) * (c // groups)
    count = count.clamp(min=1)[:, None, None, None]
    weight, bias = s["weight"].detach(), s["bias"].detach()

    def total(v):  # over an utterance's frames and a group's channels
        return v.view(n, t, groups, c // groups).sum((1, 3), keepdim=True)

    def spread(v):
        return v.expand(n, 1, groups, c // groups).reshape(n, 1, c)

    d = x - spread(total(x) / count)
    if live is not None:
        d = torch.where(live, d, 0.0)
    rstd = spread(1 / torch.sqrt(total(d * d) / count + _EPS))
    xhat = d * rstd
    a, slope = _act(xhat * weight + bias, case["act"])
    out = {"y": (a if live is None else torch.where(live, a, 0.0)).to(s["x"].dtype)}
    if not case["train"]:
        return out
    gz = s["grad_y"].float() * slope
    if live is not None:
        gz = torch.where(live, gz, 0.0)
    gxhat = gz * weight
    gx = rstd * (gxhat - spread(total(gxhat) / count) - xhat * spread(total(gxhat * xhat) / count))
    if live is not None:
        gx = torch.where(live, gx, 0.0)
    out["grad_x"] = gx.to(s["x"].dtype)
    out["grad_weight"], out["grad_bias"] = (gz * xhat).sum((0, 1)), gz.sum((0, 1))
    return out


def _philox(counters, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3): (count, 4) words."""
    low = 0xFFFFFFFF
    c0, c1 = counters & low, counters >> 32
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64, which keeps all 64 bits of the products
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), 1)


def _plain_dropout(s):
    case, x = s["case"], s["x"].detach()
    words = _philox(torch.arange((x.numel() + 3) // 4, device="cuda"), s["seed"]).view(-1)[: x.numel()].view(x.shape)
    keep, scale = words >= round(case["p"] * 2 ** 32), 1 / (1 - case["p"])
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    out = {"y": y.to(x.dtype)}
    if case["train"]:
        out["grad_x"] = torch.where(keep, s["grad_y"].float() * scale, 0.0).to(x.dtype)
        if s["residual"] is not None:
            out["grad_residual"] = s["grad_y"]
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"recurrence": _plain_recurrence, "norm": _plain_norm, "dropout": _plain_dropout}[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------


def _exact_recurrence(s):
    """Frame by frame, as the formula reads."""
    case = s["case"]
    n, t, c = case["n"], case["t"], case["c"]
    lens = torch.tensor(_lengths(case), device="cuda")[:, None]
    x, gate = (s["x"][..., :c], s["x"][..., c:]) if s["gate"] is None else (s["x"], s["gate"])
    x, gate = x.detach().double(), gate.detach().double()
    f = torch.sigmoid(gate)
    h = s["initial"].detach().double() if s["initial"] is not None else torch.zeros(n, c, device="cuda", dtype=torch.double)
    y, before = torch.zeros_like(x), torch.zeros_like(x)
    order = list(range(t - 1, -1, -1)) if case["reverse"] else list(range(t))
    for i in order:
        before[:, i] = h
        h = torch.where(i < lens, h + (1 - f[:, i]) * (x[:, i] - h), h)
        y[:, i] = torch.where(i < lens, h, 0.0)
    out = {"y": y, "final": h}
    if not case["train"]:
        return out
    m, gx, gg = s["grad_final"].double(), torch.zeros_like(x), torch.zeros_like(x)
    for i in reversed(order):
        gh = s["grad_y"][:, i].double() + m
        gx[:, i] = torch.where(i < lens, (1 - f[:, i]) * gh, 0.0)
        gg[:, i] = torch.where(i < lens, f[:, i] * (1 - f[:, i]) * gh * (before[:, i] - x[:, i]), 0.0)
        m = torch.where(i < lens, f[:, i] * gh, m)
    if s["gate"] is None:
        out["grad_x"] = torch.cat((gx, gg), 2)
    else:
        out["grad_x"], out["grad_gate"] = gx, gg
    if s["initial"] is not None:
        out["grad_initial"] = m
    return out


def _exact_norm(s):
    """Utterance by utterance and the chain rule by hand, on the frames there are."""
    case, groups = s["case"], s["case"]["groups"]
    c, per = case["c"], case["c"] // case["groups"]
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    y = torch.zeros_like(s["x"].detach(), dtype=torch.double)
    gx, gw, gb = torch.zeros_like(y), torch.zeros_like(w), torch.zeros_like(b)
    for i, length in enumerate(_lengths(case)):
        if not length:
            continue
        x = s["x"][i, :length].detach().double().view(length, groups, per)
        mean = x.mean((0, 2), keepdim=True)
        rstd = ((x - mean).square().mean((0, 2), keepdim=True) + _EPS).rsqrt()
        xhat = (x - mean) * rstd
        z = xhat.view(length, c) * w + b
        if case["act"] == "none":
            a, slope = z, torch.ones_like(z)
        elif case["act"] == "relu":
            a, slope = z.clamp(min=0), torch.heaviside(z, torch.zeros_like(z))
        elif case["act"] == "silu":
            a, slope = z * torch.sigmoid(z), torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
        else:
            cdf = (1 + _erf(z / math.sqrt(2))) / 2
            a, slope = z * cdf, cdf + z * (-z.square() / 2).exp() / math.sqrt(2 * math.pi)
        y[i, :length] = a
        if case["train"]:
            gz = s["grad_y"][i, :length].double() * slope
            gw += (gz * xhat.view(length, c)).sum(0)
            gb += gz.sum(0)
            q = (gz * w).view(length, groups, per)
            gx[i, :length] = (rstd * (q - q.mean((0, 2), keepdim=True)
                                      - xhat * (q * xhat).mean((0, 2), keepdim=True))).view(length, c)
    return {"y": y, "grad_x": gx, "grad_weight": gw, "grad_bias": gb} if case["train"] else {"y": y}


def _exact_dropout(s):
    """The generator on the host, in unsigned 64-bit arithmetic."""
    case, x = s["case"], s["x"].detach()
    count, low, half = (x.numel() + 3) // 4, np.uint64(0xFFFFFFFF), np.uint64(32)
    word = [np.arange(count, dtype=np.uint64) & low, np.arange(count, dtype=np.uint64) >> half,
            np.zeros(count, np.uint64), np.zeros(count, np.uint64)]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * word[0], np.uint64(0xCD9E8D57) * word[2]
        word = [(b >> half) ^ word[1] ^ np.uint64(key[0]), b & low, (a >> half) ^ word[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    dropped = np.stack(word, 1).reshape(-1)[: x.numel()] < np.uint64(math.floor(case["p"] * 2 ** 32 + 0.5))
    keep = ~torch.from_numpy(dropped).cuda().view(x.shape)
    y = keep * x.double() / (1 - case["p"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().double()
    out = {"y": y}
    if case["train"]:
        out["grad_x"] = keep * s["grad_y"].double() / (1 - case["p"])
        if s["residual"] is not None:
            out["grad_residual"] = s["grad_y"].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "norm": _exact_norm, "dropout": _exact_dropout}[case["op"]](s)
