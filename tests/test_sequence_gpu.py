"""The sequence operators (``sequence.py``) on the GPU, against the float64 restatement in ``oracle/sequence_oracle.py``.

Tolerances: the restatement's own error bound for float32 (float64) arithmetic, plus half a step of the output's type
relative to the value.  Frames behind an utterance's end hold NaN, infinities and the type's lowest value in every test
with lengths: they must not be seen.
"""
import numpy as np
import pytest
import torch

import capi
import sequence
from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps for t in TYPES}  # half a step below the normal range


def _unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, pair, dtype, name):
    value, bound = pair
    got = _np(got)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    if not value.size:
        return
    allowed = bound + HALF_STEP[dtype] * (np.abs(value) + bound) + TINY[dtype]
    excess = np.abs(got - value) - allowed
    assert np.isfinite(got).all(), name
    worst = np.unravel_index(np.argmax(excess), excess.shape)
    assert excess[worst] <= 0, (name, worst, got[worst], value[worst], allowed[worst])


def _poison(t, lens):
    """What must never be seen, behind the end of each utterance."""
    bad = [float("nan"), float("inf"), float("-inf"), torch.finfo(t.dtype).min]
    for i, length in enumerate(lens):
        for j in range(max(int(length), 0), t.shape[1]):
            t[i, j] = bad[j % 4]
    return t


def _laid_out(t, layout):
    """The same values: as they are, time-major, channels of a wider tensor, or off the 16-byte grid."""
    n, f, c = t.shape
    if layout == "time-major":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if layout == "wide":
        wide = torch.full((n, f, 2 * c + 8), float("nan"), dtype=t.dtype, device=t.device)
        wide[..., 8:8 + c] = t
        return wide[..., 8:8 + c]
    if layout == "odd":
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(n, f, c)
    if layout == "channels apart":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    return t


# ---- gated recurrence ------------------------------------------------------------------------------------------------

# (batch, frames, channels, lens, reverse, with an initial state, layout)
RECURRENCES = [
    (1, 1, 1, None, False, False, "dense"),
    (3, 1, 70, None, False, True, "packed"),
    (2, 2, 8, [2, 1], True, True, "dense"),
    (4, 15, 33, [15, 0, 7, 1], False, True, "packed"),
    (4, 16, 64, [16, 0, 15, 1], True, False, "packed"),
    (3, 17, 32, [17, 16, 0], False, False, "time-major"),
    (2, 33, 128, None, True, True, "wide"),
    (2, 63, 40, [63, 64 + 5], False, True, "odd"),
    (2, 64, 96, [-3, 40], True, True, "time-major"),
    (3, 65, 24, [65, 64, 63], False, False, "channels apart"),
    (2, 130, 256, [129, 128], True, True, "packed"),
    (5, 257, 31, [257, 256, 255, 0, 129], False, True, "packed"),
    (1, 1031, 16, None, True, False, "packed"),
    (2, 700, 72, [513, 700], False, True, "dense"),
    (1, 5000, 8, None, False, True, "packed"),
    (70, 9, 48, [i % 10 for i in range(70)], True, False, "packed"),
    (3, 140, 34, [140, 139, 7], True, True, "dense"),
    (2, 300, 50, None, False, True, "packed"),
    (40, 300, 130, [300 - 7 * i for i in range(40)], False, True, "time-major"),
    (33, 600, 160, [600] * 16 + [i for i in range(17)], True, False, "packed"),
]


def _recurrence_problem(case, dtype, seed):
    n, t, c, lens, reverse, with_initial, layout = case
    rng = np.random.default_rng(seed)

    def tensor(*shape, mean=0.0, to=dtype):
        return torch.from_numpy(rng.standard_normal(shape) + mean).to("cuda").to(to)

    state = torch.float64 if dtype == torch.float64 else torch.float32
    p = {"x": tensor(n, t, c), "gate": tensor(n, t, c, mean=1.0).clamp(-8, 8), "grad_y": tensor(n, t, c),
         "grad_final": tensor(n, c, to=state), "initial": tensor(n, c, to=state) if with_initial else None}
    want = so.recurrence(*(_np(p[k]) if p[k] is not None else None for k in ("x", "gate", "initial")), lens, reverse,
                         _np(p["grad_y"]), _np(p["grad_final"]), _unit(dtype))
    if lens is not None:
        for k in ("x", "gate", "grad_y"):
            _poison(p[k], lens)
    p["lens"] = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    return p, want


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", RECURRENCES, ids=lambda c: "%dx%dx%d-%s" % (c[0], c[1], c[2], c[6]))
def test_recurrence(case, dtype):
    n, t, c, lens, reverse, with_initial, layout = case
    p, want = _recurrence_problem(case, dtype, 7 * n + 11 * t + c)
    leaves = []
    if layout == "packed":
        x, gate = torch.cat((p["x"], p["gate"]), 2).requires_grad_(True), None
        leaves.append(x)
    else:
        x, gate = (_laid_out(p[k], layout).detach().requires_grad_(True) for k in ("x", "gate"))
        leaves += [x, gate]
    initial = p["initial"]
    if with_initial:
        leaves.append(initial.requires_grad_(True))
    grad_y = _laid_out(p["grad_y"], layout)
    runs = []
    for _ in range(2):
        y, final = sequence.gated_recurrence(x, gate, initial, p["lens"], reverse)
        runs.append([y, final] + list(torch.autograd.grad([y, final], leaves, [grad_y, p["grad_final"]])))
    assert all(torch.equal(a, b) for a, b in zip(*runs)), "two runs differ"
    y, final, *grads = runs[0]
    assert y.dtype == dtype and final.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    _close(y, want["y"], dtype, "y")
    _close(final, want["final"], final.dtype, "final")
    if layout == "packed":
        grads[:1] = [grads[0][..., :c], grads[0][..., c:]]
    _close(grads[0], want["grad_x"], dtype, "grad_x")
    _close(grads[1], want["grad_gate"], dtype, "grad_gate")
    if with_initial:
        _close(grads[2], want["grad_initial"], final.dtype, "grad_initial")
    if layout == "time-major" and n > 1 and t > 1:
        assert y.transpose(0, 1).is_contiguous()
    # without a graph: the same values from the call that keeps no states
    with torch.no_grad():
        y2, final2 = sequence.gated_recurrence(x, gate, initial, p["lens"], reverse)
    assert torch.equal(y2, y) and torch.equal(final2, final)


def test_recurrence_in_pieces():
    """A stream fed in pieces with the state carried is the stream fed at once (the state is not rounded to 16 bits)."""
    case = (3, 200, 40, None, False, True, "dense")
    p, want = _recurrence_problem(case, torch.bfloat16, 5)
    state, parts, at = p["initial"], [], 0
    for size in [1, 1, 1, 16, 30, 1, 100, 50]:
        y, state = sequence.gated_recurrence(p["x"][:, at:at + size], p["gate"][:, at:at + size], state)
        parts.append(y)
        at += size
    assert at == 200
    _close(torch.cat(parts, 1), want["y"], torch.bfloat16, "y")
    _close(state, want["final"], torch.float32, "final")


def test_recurrence_extreme_gates():
    """Gates that are shut or open for good, in the type's whole range: no NaN, and exactly the kept or the new value."""
    for dtype in TYPES:
        top = torch.finfo(dtype).max
        gate = torch.tensor([top, -top, float("inf"), float("-inf"), 200.0, -200.0], device="cuda", dtype=dtype)
        gate = gate.repeat(40).view(1, -1, 1).expand(1, 240, 8).contiguous()
        x = torch.arange(1, 241, device="cuda", dtype=dtype).view(1, -1, 1).expand(1, 240, 8).contiguous().requires_grad_(True)
        y, final = sequence.gated_recurrence(x, gate.requires_grad_(True))
        # odd frames take their value, even ones keep the state
        want = torch.arange(1, 241).view(-1, 2)[:, 0] - 1
        assert torch.equal(y[0, :, 0].double().cpu(), torch.stack((want, want + 2), 1).view(-1).to(dtype).double()), dtype
        gx, gg = torch.autograd.grad([y.sum() + final.sum()], [x, gate])
        # f (1 - f) is at most the least sigmoid there is: 2^-126 = 1.2e-38 in float32 arithmetic, exp(-200) = 1.4e-87 in
        # float64; times |h - x| and the gradient's sum, each at most 480
        least = 1.4e-87 if dtype == torch.float64 else 2.0 ** -126
        assert torch.isfinite(gx).all() and float(gg.abs().max()) <= 1.01 * least * 480 * 480


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
def test_recurrence_sigmoid_and_its_complement(dtype):
    """Gates up to +-80, one frame: behind a state of 1 and a value of 0 the output is sigmoid(gate), the other way round its
    complement, each to the step's bound relative to itself (1e-35 at the far end)."""
    gate = torch.linspace(-80, 80, 200001, device="cuda", dtype=torch.float64).to(dtype).view(1, 1, -1)
    g, u = _np(gate)[0, 0], _unit(dtype)
    zero, one = torch.zeros_like(gate), torch.ones_like(gate)
    f, _ = sequence.gated_recurrence(zero, gate, one[:, 0])
    keep, _ = sequence.gated_recurrence(one, gate, zero[:, 0])
    for got, want in ((f, so.sigmoid(g)), (keep, so.sigmoid(-g))):
        assert (np.abs(_np(got)[0, 0] - want) <= so.gate_step(g) * u * want).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,t,c,reverse", [(3, 4, 10, False), (2, 150, 33, True), (2, 150, 64, False), (2, 700, 16, True)])
def test_recurrence_gates_up_to_80(n, t, c, reverse, dtype):
    rng = np.random.default_rng(t + c)
    state = torch.float64 if dtype == torch.float64 else torch.float32
    x, gate, gy = (torch.from_numpy(v).to("cuda").to(dtype) for v in
                   (rng.standard_normal((n, t, c)), rng.uniform(-80, 80, (n, t, c)), rng.standard_normal((n, t, c))))
    initial, gf = (torch.from_numpy(rng.standard_normal((n, c))).to("cuda").to(state) for _ in range(2))
    want = so.recurrence(_np(x), _np(gate), _np(initial), None, reverse, _np(gy), _np(gf), _unit(dtype))
    leaves = [v.requires_grad_(True) for v in (x, gate, initial)]
    y, final = sequence.gated_recurrence(*leaves, reverse=reverse)
    grads = torch.autograd.grad([y, final], leaves, [gy, gf])
    for got, name in zip((y, final) + grads, ("y", "final", "grad_x", "grad_gate", "grad_initial")):
        _close(got, want[name], state if name in ("final", "grad_initial") else dtype, name)


@pytest.mark.parametrize("frames", [3, 40, 600])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64], ids=str)
def test_recurrence_shut_gate_behind_a_huge_state(frames, dtype):
    """A gate of -infinity (or the type's lowest value, or far enough below zero) takes its frame's value alone, whatever
    finite value the state had; and its gradient passes nothing back."""
    huge = torch.finfo(dtype).min
    x = torch.ones(2, frames, 8, device="cuda", dtype=dtype)
    x[:, ::2] = huge
    # -200: exp(-200) is 0 beside any float, and 1e-87 in double, where a huge state would show
    shut = [float("-inf"), torch.finfo(dtype).min, -1e5, -200.0 if dtype != torch.float64 else -1e5]
    gate = torch.tensor(shut * 2, device="cuda", dtype=dtype).expand(2, frames, 8).contiguous()
    x.requires_grad_(True), gate.requires_grad_(True)
    initial = torch.full((2, 8), torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).min, device="cuda",
                         dtype=torch.float64 if dtype == torch.float64 else torch.float32, requires_grad=True)
    for reverse in (False, True):
        y, final = sequence.gated_recurrence(x, gate, initial, reverse=reverse)
        assert torch.equal(y, x)
        gx, gg, gi = torch.autograd.grad([y, final], [x, gate, initial], [torch.ones_like(y), torch.zeros_like(final)])
        assert torch.equal(gx, torch.ones_like(gx)) and not gg.any() and not gi.any()


def test_recurrence_strides_beyond_32_bits():
    """Frames 2^30 elements apart: the offsets pass 32 bits."""
    flat = torch.zeros(5 * 2 ** 30 + 64, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((1, 6, 32), (0, 2 ** 30, 1))
    gate = flat[32:].as_strided((1, 6, 32), (0, 2 ** 30, 1))
    small = torch.randn(1, 6, 32, device="cuda").bfloat16(), torch.randn(1, 6, 32, device="cuda").bfloat16()
    x.copy_(small[0])
    gate.copy_(small[1])
    got, want = sequence.gated_recurrence(x, gate), sequence.gated_recurrence(*small)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("reverse", [False, True])
def test_recurrence_frames_2_to_31_apart(reverse):
    """Frames beyond what a 32-bit step reaches: the form of one thread per channel, both ways."""
    far, dtype = 2 ** 31, torch.bfloat16
    flat = torch.empty(4 * far + 96, dtype=dtype, device="cuda")
    rng = np.random.default_rng(17)
    small = [torch.from_numpy(rng.standard_normal((1, 5, 32))).to("cuda").to(dtype) for _ in range(3)]
    x, gate, gy = (flat[32 * k:].as_strided((1, 5, 32), (0, far, 1)) for k in range(3))
    for v, w in zip((x, gate, gy), small):
        v.copy_(w)
    initial, gf = (torch.from_numpy(rng.standard_normal((1, 32))).to("cuda").float() for _ in range(2))
    want = so.recurrence(*(_np(v) for v in (small[0], small[1], initial)), None, reverse, _np(small[2]), _np(gf))
    leaves = [v.detach().requires_grad_(True) for v in (x, gate, initial)]
    y, final = sequence.gated_recurrence(*leaves, reverse=reverse)
    grads = torch.autograd.grad([y, final], leaves, [gy, gf])
    for got, name in zip((y, final) + grads, ("y", "final", "grad_x", "grad_gate", "grad_initial")):
        _close(got, want[name], torch.float32 if name in ("final", "grad_initial") else dtype, name)


def test_recurrence_empty():
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = torch.randn(*shape, device="cuda", requires_grad=True)
        gate = torch.randn(*shape, device="cuda", requires_grad=True)
        initial = torch.randn(shape[0], shape[2], device="cuda", requires_grad=True)
        y, final = sequence.gated_recurrence(x, gate, initial)
        assert y.shape == shape and torch.equal(final, initial)
        grads = torch.autograd.grad(y.sum() + 2 * final.sum(), [x, gate, initial])
        assert torch.equal(grads[0], torch.zeros_like(x)) and (shape[1] or torch.equal(grads[2], torch.full_like(initial, 2)))


def test_recurrence_gradients_of_one_output_and_broadcast():
    """Only one output used; an expanded input, an expanded gradient."""
    gate = torch.randn(2, 20, 8, device="cuda", dtype=torch.float64, requires_grad=True)
    row = torch.randn(1, 1, 8, device="cuda", dtype=torch.float64, requires_grad=True)
    for pick in (lambda y, final: y.sum(), lambda y, final: final.sum()):
        got = torch.autograd.grad(pick(*sequence.gated_recurrence(row.expand(2, 20, 8), gate)), [row, gate])
        full = row.detach().expand(2, 20, 8).contiguous().requires_grad_(True)
        want = torch.autograd.grad(pick(*sequence.gated_recurrence(full, gate)), [full, gate])
        assert torch.allclose(got[0], want[0].sum((0, 1), keepdim=True), rtol=1e-13, atol=0) and torch.equal(got[1], want[1])


# ---- group norm with an activation -----------------------------------------------------------------------------------

# (batch, frames, channels, groups, lens, activation, with parameters, layout)
NORMS = [
    (1, 1, 1, 1, None, "none", True, "dense"),
    (2, 1, 64, 8, None, "relu", True, "dense"),
    (300, 1, 96, 4, None, "silu", True, "dense"),
    (3, 5, 12, 3, [5, 0, 1], "gelu", True, "dense"),
    (2, 41, 256, 8, None, "relu", True, "dense"),
    (4, 33, 66, 11, [33, 0, 32, 7], "silu", True, "odd"),
    (2, 64, 128, 1, [40, 64], "gelu", False, "time-major"),
    (2, 65, 128, 128, [65, 64], "none", True, "wide"),
    (3, 130, 330, 11, [129, -1, 130], "gelu", True, "dense"),
    (2, 200, 1024, 32, [200, 77], "relu", True, "dense"),
    (2, 100, 72, 2, None, "silu", True, "channels apart"),
    (1, 1500, 40, 5, [1499], "silu", True, "dense"),
    (1, 3001, 512, 2, None, "gelu", True, "wide"),
    (2, 500, 256, 1, [500, 490], "silu", True, "dense"),
    (2, 900, 256, 1, None, "relu", True, "dense"),
    (2, 100, 256, 1, [100, 3], "none", True, "odd"),
    (3, 20, 1200, 1, None, "silu", True, "dense"),
    (3, 20, 1200, 1, [20, 0, 19], "gelu", True, "odd"),
    (2, 5, 4100, 1, None, "silu", True, "odd"),
    (2500, 1, 32, 4, None, "relu", True, "dense"),
    (1100, 2, 10, 5, [i % 3 for i in range(1100)], "silu", True, "time-major"),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "%dx%dx%d-%d-%s-%s" % (c[0], c[1], c[2], c[3], c[5], c[7]))
def test_group_norm_act(case, dtype):
    n, t, c, groups, lens, act, affine, layout = case
    rng = np.random.default_rng(13 * n + 5 * t + c)
    state = torch.float64 if dtype == torch.float64 else torch.float32
    x = torch.from_numpy(rng.standard_normal((n, t, c)) * 1.5 + 0.5).to("cuda").to(dtype)
    grad_y = torch.from_numpy(rng.standard_normal((n, t, c))).to("cuda").to(dtype)
    weight = bias = None
    if affine:
        weight = torch.from_numpy(1 + 0.3 * rng.standard_normal(c)).to("cuda").to(state).requires_grad_(True)
        bias = torch.from_numpy(0.3 * rng.standard_normal(c)).to("cuda").to(state).requires_grad_(True)
    want = so.group_norm_act(_np(x), groups, None if weight is None else _np(weight), None if bias is None else _np(bias),
                             lens, 1e-5, act, _np(grad_y), _unit(dtype))
    if lens is not None:
        _poison(x, lens), _poison(grad_y, lens)
    x, grad_y = _laid_out(x, layout).detach().requires_grad_(True), _laid_out(grad_y, layout)
    lens_d = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    leaves = [x] + ([weight, bias] if affine else [])
    runs = []
    for _ in range(2):
        y = sequence.group_norm_act(x, groups, weight, bias, lens_d, 1e-5, act)
        runs.append([y] + list(torch.autograd.grad(y, leaves, grad_y)))
    assert all(torch.equal(a, b) for a, b in zip(*runs)), "two runs differ"
    y, gx, *grads = runs[0]
    assert y.dtype == dtype
    _close(y, want["y"], dtype, "y")
    _close(gx, want["grad_x"], dtype, "grad_x")
    if affine:
        _close(grads[0], want["grad_weight"], state, "grad_weight")
        _close(grads[1], want["grad_bias"], state, "grad_bias")
    with torch.no_grad():
        assert torch.equal(sequence.group_norm_act(x, groups, weight, bias, lens_d, 1e-5, act), y)


def test_relu_slope_at_the_training_size():
    """32 utterances of 200 to 800 frames and 1024 channels: every gradient against float64, and every side of ReLU's corner
    that is not the one of 64 bits lies within float32's rounding of it.

    z = (x - mean) * (rstd * weight) + bias: near the corner the two terms are as large as the bias.  mean is off by a few
    units of the values (2^-24 * 0.5), rstd by a few of its own, the factor and the product by half a unit each: below 16
    units of |bias| + |mean * rstd * weight|, some 2e-6.  With grad_y zero wherever |z| is below that no gradient depends on
    the side, and what is left is rounding: single terms to 16 units, sums of up to 25600 terms by trees."""
    n, t, c, groups = 32, 800, 1024, 32
    lens = torch.tensor([200 + 600 * (7 * i % 32) // 31 for i in range(n)], dtype=torch.int32, device="cuda")
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(n, t, c, device="cuda", generator=gen).mul_(1.5).add_(0.5)
        w = torch.randn(c, device="cuda", generator=gen).mul_(0.2).add_(1)
        b = torch.randn(c, device="cuda", generator=gen).mul_(0.2)
        gy = torch.randn(n, t, c, device="cuda", generator=gen)
        wd, bd = w.double(), b.double()
        y = sequence.group_norm_act(x, groups, w, b, lens)
        want = [torch.zeros(n, t, c, device="cuda", dtype=torch.float64)] + [torch.zeros_like(wd) for _ in range(2)]
        for i in range(n):
            length = int(lens[i])
            v = x[i, :length].double().view(length, groups, -1)
            mean = v.mean((0, 2), keepdim=True)
            rstd = ((v - mean).square().mean((0, 2), keepdim=True) + 1e-5).rsqrt()
            xhat = ((v - mean) * rstd).view(length, c)
            z = xhat * wd + bd
            around = (mean.abs() * rstd).expand(1, groups, c // groups).reshape(c) * wd.abs() + bd.abs()
            near = z.abs() <= 16 * 2 ** -24 * around
            assert not bool((((y[i, :length] > 0) != (z > 0)) & ~near).any())
            gy[i, :length].masked_fill_(near, 0)
            gz = gy[i, :length].double() * (z > 0)
            want[1] += (gz * xhat).sum(0)
            want[2] += gz.sum(0)
            q, h = (gz * wd).view(length, groups, -1), xhat.view(length, groups, -1)
            want[0][i, :length] = (rstd * (q - q.mean((0, 2), keepdim=True) - h * (q * h).mean((0, 2), keepdim=True))).view(length, c)
        leaves = [v.requires_grad_(True) for v in (x, w, b)]
        got = torch.autograd.grad(sequence.group_norm_act(x, groups, w, b, lens), leaves, gy)
        for g, ref in zip(got, want):
            assert float((g - ref).norm() / ref.norm()) <= 1e-6


def test_group_norm_large_mean():
    """Values far from zero: the variance is taken from deviations, not as a difference of squares.

    x = 4096 + z in float32 is exact to 2^-12; the deviations' relative error is about 2^-12 at worst from the mean's
    rounding (2^-12 absolute), which moves every value alike and leaves the variance at 2^-24 relative."""
    z = torch.randn(2, 300, 64, device="cuda", dtype=torch.float64)
    x = (z + 4096).float()
    y = sequence.group_norm_act(x, 8, activation="none").double()
    d = x.double().view(2, 300, 8, 8)
    want = ((d - d.mean((1, 3), keepdim=True)) / (d.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()).view_as(x)
    assert float((y - want).abs().max()) <= 2 ** -10
    assert abs(float(y.var(unbiased=False)) - 1) <= 1e-3


@pytest.mark.parametrize("frames,channels", [(1, 8), (40, 64), (3000, 512)])
def test_group_norm_beyond_the_statistics_range(frames, channels):
    """Squares that pass float32 leave no variance of zero behind: |(x - mean) / std| of n values is at most sqrt(n), so
    nothing finite may be larger.  The other groups do not notice."""
    x = torch.randn(2, frames, channels, device="cuda")
    per = channels // 2
    wild = x.clone()
    wild[1, :, per:] *= 3e30
    y, want = (sequence.group_norm_act(v, 2, activation="none") for v in (wild, x))
    assert torch.equal(y[0], want[0]) and torch.equal(y[1, :, :per], want[1, :, :per])
    off = y[1, :, per:]
    assert not bool((off.abs() > (frames * per) ** 0.5 * (1 + 1e-5)).any())


@pytest.mark.parametrize("frames,channels,std", [(1, 8, 1e17), (5, 64, 1e17), (40, 64, 1e17), (700, 256, 1e16), (3000, 512, 1e16)])
def test_group_norm_far_mean_within_the_range(frames, channels, std):
    """Values about 1e20, whose squares pass float32 while their squared deviations do not: in the forms that one team, a
    block, a cluster and two launches have.

    The mean of values of one size is off by at most 16 of its units (a few joins and a short tree), that is 16 * 2^-24 * 1e20
    / std of a standard deviation; the normalised values move by that much alike, the variance by its square, and float32
    rounds a few times at values below 6."""
    gen = torch.Generator(device="cuda").manual_seed(21)
    x = (1e20 + std * torch.randn(2, frames, channels, device="cuda", dtype=torch.float64, generator=gen)).float()
    grad = torch.randn(2, frames, channels, device="cuda", generator=gen)
    want = so.group_norm_act(_np(x), 2, act="none", grad_y=_np(grad))
    x.requires_grad_(True)
    y = sequence.group_norm_act(x, 2, activation="none")
    _close(y, want["y"], torch.float32, "y")
    off = 16 * 2 ** -24 * 1e20 / std
    assert np.abs(_np(y) - want["y"][0]).max() <= off + 6 * off ** 2 + 64 * 2 ** -24
    _close(torch.autograd.grad(y, x, grad)[0], want["grad_x"], torch.float32, "grad_x")


@pytest.mark.parametrize("value", [1e19, -3e19, 1e30, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("frames,channels", [(1, 8), (40, 64), (3000, 512)])
def test_group_norm_of_one_value(frames, channels, value):
    """A group that holds one value throughout, up to the type's lowest: sums of the values pass the type, the mean does not.
    The normalised values are the mean's rounding over itself at most, never NaN."""
    x = torch.full((2, frames, channels), value, device="cuda", requires_grad=True)
    y = sequence.group_norm_act(x, 2, activation="none")
    assert torch.isfinite(y).all() and torch.isfinite(torch.autograd.grad(y.sum(), x)[0]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_silu_far_below_zero(dtype):
    """SiLU and its slope are nothing at z = -200 and below, down to the type's lowest value and -infinity: at most
    128 * 2^-126 = 1.6e-36 in float32 arithmetic.  The other channels do not notice."""
    state = torch.float64 if dtype == torch.float64 else torch.float32
    lowest = torch.finfo(state).min
    for frames in (3, 40, 3000):
        x = torch.randn(2, frames, 512, device="cuda").to(dtype).requires_grad_(True)
        bias = torch.zeros(512, dtype=state, device="cuda")
        plain = sequence.group_norm_act(x, 2, None, bias, activation="silu")
        bias[::8] = torch.tensor([-200.0, -1e10, -1e30, -1e37, lowest / 2, lowest, float("-inf"), -1e35], device="cuda",
                                 dtype=state).repeat(8)
        bias.requires_grad_(True)
        y = sequence.group_norm_act(x, 2, None, bias, activation="silu")
        far = torch.zeros(512, dtype=torch.bool, device="cuda")
        far[::8] = True
        assert float(y[..., far].detach().abs().max()) <= 1.6e-36 and torch.equal(y[..., ~far], plain[..., ~far])
        grad = torch.zeros_like(y)
        grad[..., far] = 1
        gx, gb = torch.autograd.grad(y, [x, bias], grad)
        # slopes below 1.6e-36, summed over at most 2 x 3000 frames, times 1 / std = 1 for the input's gradient
        assert float(gb.abs().max()) <= 6000 * 1.6e-36 and float(gx.abs().max()) <= 6000 * 1.6e-36


def test_group_norm_other_shapes():
    """(batch, channels), images channels last, 16-bit parameters, no frames, no utterances."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 64, device="cuda", generator=gen)
    assert torch.equal(sequence.group_norm_act(x, 4, activation="silu"),
                       sequence.group_norm_act(x.view(5, 1, 64), 4, activation="silu").view(5, 64))
    image = torch.randn(2, 32, 9, 11, device="cuda", generator=gen).to(memory_format=torch.channels_last)
    y = sequence.group_norm_act(image.permute(0, 2, 3, 1), 4, activation="relu")
    want = so.group_norm_act(_np(image.permute(0, 2, 3, 1).reshape(2, 99, 32)), 4, act="relu")["y"]
    _close(y.reshape(2, 99, 32), want, torch.float32, "image")
    w = (1 + torch.randn(64, device="cuda", generator=gen)).bfloat16().requires_grad_(True)
    x16 = x.bfloat16().requires_grad_(True)
    y = sequence.group_norm_act(x16, 4, w)
    assert torch.equal(y, sequence.group_norm_act(x16, 4, w.float()))
    gw, = torch.autograd.grad(y.sum(), [w])
    assert gw.dtype == torch.bfloat16
    for shape in ((0, 5, 8), (2, 0, 8)):
        e = torch.randn(*shape, device="cuda", requires_grad=True)
        weight, bias = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
        y = sequence.group_norm_act(e, 2, weight, bias)
        assert y.shape == shape
        grads = torch.autograd.grad(y.sum(), [e, weight, bias])
        assert all(torch.equal(g, torch.zeros_like(g)) for g in grads)


def test_many_utterances():
    """More utterances than a grid's second extent has blocks, and than fit one block's run: the same bits as in pieces."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(140001, 1, 16, device="cuda", generator=gen, requires_grad=True)
    gy = torch.randn(140001, 1, 16, device="cuda", generator=gen)
    w = torch.randn(16, device="cuda", generator=gen, requires_grad=True)
    y = sequence.group_norm_act(x, 2, w, activation="silu")
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    want_w = torch.zeros(16, dtype=torch.float64, device="cuda")
    for part in range(0, 140001, 40000):
        piece = x.detach()[part:part + 40000].requires_grad_(True)
        z = sequence.group_norm_act(piece, 2, w, activation="silu")
        g, v = torch.autograd.grad(z, [piece, w], gy[part:part + 40000])
        assert torch.equal(z, y[part:part + 40000]) and torch.equal(g, gx[part:part + 40000])
        want_w += v
    # sums of 140001 terms of order one in float32, in other groupings: 2^-24 * 140001 relative to the terms' sum at worst
    assert float((gw - want_w).abs().max()) <= 140001 * 2 ** -24 * 140001 ** 0.5 * 4
    h, _ = sequence.gated_recurrence(x.detach().expand(140001, 9, 16), gy.expand(140001, 9, 16))
    h2, _ = sequence.gated_recurrence(x.detach()[139000:].expand(1001, 9, 16), gy[139000:].expand(1001, 9, 16))
    assert torch.equal(h[139000:], h2)


def test_parameter_sums_of_many_utterances():
    """Parameter gradients over more utterances than a grid's second extent has blocks, against float64.

    Rounding: a channel's sum wanders within some sqrt(140001) = 374 (terms of order one, either sign), rounded at most 300
    times on the way of one value (the utterances a block takes, the sets, the join): 2^-24 * 374 * sqrt(300) = 4e-4; the
    terms themselves are off by some 8 units each: 8 * 2^-24 * 374 = 2e-4.  1e-2 leaves a factor of 16; a single utterance that
    is lost or taken twice moves the 16 channels by terms of order one (checked for a few of them)."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    n, c = 140001, 16
    x, gy = (torch.randn(n, 1, c, device="cuda", generator=gen) for _ in range(2))
    w, b = (torch.randn(c, device="cuda", generator=gen) for _ in range(2))
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    got = torch.autograd.grad(sequence.group_norm_act(x, 2, w, b, activation="silu"), leaves, gy)
    v = x.detach().double().view(n, 2, c // 2)
    d = v - v.mean(2, keepdim=True)
    xhat = (d / (d.square().mean(2, keepdim=True) + 1e-5).sqrt()).view(n, c)
    z = xhat * w.detach().double() + b.detach().double()
    s = torch.sigmoid(z)
    gz = gy.view(n, c).double() * s * (1 + z * (1 - s))
    for g, terms in ((got[1], gz * xhat), (got[2], gz)):
        assert float((g - terms.sum(0)).abs().max()) <= 1e-2
        assert all(float(terms[i].abs().max()) > 2e-2 for i in (0, 65534, 65535, 131070, n - 1))


def test_group_norm_statistics_beyond_2_to_31():
    """2^30 + 1024 groups of all utterances, so that the statistics have more than 2^31 elements: the last utterances get what
    they get in a call of their own, forward and backward."""
    n, c = 2 ** 20 + 1, 1024
    gen = torch.Generator(device="cuda").manual_seed(5)
    last = torch.randn(5, 2, c, device="cuda", generator=gen).bfloat16()
    x, gy = (torch.zeros(n, 2, c, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    where = [0, 524287, 524288, n - 2, n - 1]
    for i, k in enumerate(where):
        x[k], gy[k] = last[i], last[4 - i]
    x.requires_grad_(True)
    y = sequence.group_norm_act(x, c, activation="silu")
    gx, = torch.autograd.grad(y, x, gy)
    small = last.clone().requires_grad_(True)
    want = sequence.group_norm_act(small, c, activation="silu")
    want_x, = torch.autograd.grad(want, small, last.flip(0))
    assert torch.equal(y[where], want) and torch.equal(gx[where], want_x)
    assert int(torch.count_nonzero(y)) == int(torch.count_nonzero(want))


def test_group_norm_strides_beyond_32_bits():
    flat = torch.zeros(5 * 2 ** 30 + 64, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((1, 6, 32), (0, 2 ** 30, 1))
    small = torch.randn(1, 6, 32, device="cuda").bfloat16()
    x.copy_(small)
    assert torch.equal(sequence.group_norm_act(x, 4), sequence.group_norm_act(small, 4))


# ---- counter-based dropout -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,layout", [((1,), "dense"), ((3,), "dense"), ((1024,), "dense"), ((7, 13), "dense"),
                                          ((2, 33, 40), "wide"), ((4, 5, 64), "time-major"), ((3, 7, 11), "odd"),
                                          ((2, 3, 21), "wide"), ((3, 1000, 37), "dense"), ((64, 1, 512), "dense")])
def test_dropout(shape, layout, dtype):
    rng = np.random.default_rng(sum(shape))
    u = _unit(dtype)
    for p, seed, with_residual in ((0.05, 1, False), (0.5, 2 ** 63 + 12345, True), (1.0, 7, True), (0.3, -1, False)):
        x = torch.from_numpy(rng.standard_normal(shape)).to("cuda").to(dtype)
        grad_y = torch.from_numpy(rng.standard_normal(shape)).to("cuda").to(dtype)
        residual = torch.from_numpy(rng.standard_normal(shape)).to("cuda").to(dtype) if with_residual else None
        keep = so.dropout_keep(shape, p, seed & (2 ** 64 - 1))
        # what is dropped must not be seen
        x[torch.from_numpy(~keep).cuda()] = float("nan")
        scale = 1 / (1 - p) if p < 1 else 0.0
        kept = np.where(keep, np.nan_to_num(_np(x)) * scale, 0)
        value = kept + (_np(residual) if with_residual else 0)
        # the factor, the product and the sum are rounded once each
        bound = 2 * u * np.abs(kept) + u * np.abs(value)
        if len(shape) == 3:
            x, grad_y = _laid_out(x, layout), _laid_out(grad_y, layout)
            residual = _laid_out(residual, layout) if with_residual else None
        x = x.detach().requires_grad_(True)
        leaves = [x] + ([residual.requires_grad_(True)] if with_residual else [])
        y = sequence.philox_dropout(x, p, True, seed, residual)
        grads = torch.autograd.grad(y, leaves, grad_y)
        assert y.dtype == dtype and y.shape == torch.Size(shape)
        _close(y, (value, bound), dtype, "y")
        g = np.where(keep, _np(grad_y) * scale, 0)
        _close(grads[0], (g, 2 * u * np.abs(g)), dtype, "grad_x")
        if with_residual:
            assert torch.equal(grads[1], grad_y)
        by_tensor = sequence.philox_dropout(x, p, True, torch.tensor(seed if seed < 2 ** 63 else seed - 2 ** 64, device="cuda"),
                                            residual)
        assert torch.equal(by_tensor, y)


def test_dropout_evaluation_and_defaults():
    x, r = torch.randn(4, 50, device="cuda"), torch.randn(4, 50, device="cuda")
    assert sequence.philox_dropout(x, 0.5, False) is x and sequence.philox_dropout(x, 0.0) is x
    assert torch.equal(sequence.philox_dropout(x, 0.5, False, residual=r), x + r)
    torch.manual_seed(5)
    a = sequence.philox_dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(sequence.philox_dropout(x, 0.5), a) and not torch.equal(sequence.philox_dropout(x, 0.5), a)
    assert sequence.philox_dropout(torch.empty(0, 4, device="cuda"), 0.5).shape == (0, 4)
    big = torch.ones(1 << 20, device="cuda")
    kept = float((sequence.philox_dropout(big, 0.1, True, 99) != 0).float().mean())
    assert abs(kept - 0.9) <= 5 * (0.09 / (1 << 20)) ** 0.5


def test_dropout_probabilities_at_the_words_resolution():
    """Probabilities next to a whole number of 2^-32, and below one of them: the words are compared with the nearest whole
    number, the kept elements scaled by what is asked for."""
    x = torch.randn(1 << 16, device="cuda", dtype=torch.float64, requires_grad=True)
    words = so.philox4x32_10(np.arange(1 << 14), 5).reshape(-1)
    at = float(int(words[1000]))  # a word that lies on the border
    for p in (1e-11, 2.0 ** -34, at * 2.0 ** -32, (at + 0.49) * 2.0 ** -32, (at + 0.51) * 2.0 ** -32, 1 - 2.0 ** -40):
        keep = so.dropout_keep((1 << 16,), p, 5)
        y = sequence.philox_dropout(x, p, True, 5)
        g, = torch.autograd.grad(y.sum(), x)
        for got, ref in ((y, np.where(keep, _np(x) / (1 - p), 0)), (g, keep / (1 - p))):
            assert (np.abs(_np(got) - ref) <= 2 * 2.0 ** -53 * np.abs(ref)).all(), p
    assert so.dropout_keep((1 << 16,), at * 2.0 ** -32, 5)[1000] and not so.dropout_keep((1 << 16,), (at + 0.51) * 2.0 ** -32, 5)[1000]


def test_dropout_seed_under_a_default_device():
    """The seed comes from the CPU generator whatever device new tensors go to."""
    x = torch.randn(4, 50, device="cuda")
    torch.manual_seed(5)
    want = sequence.philox_dropout(x, 0.5)
    torch.manual_seed(5)
    with torch.device("cuda"):
        assert torch.equal(sequence.philox_dropout(x, 0.5), want)


def test_dropout_offsets_beyond_32_bits():
    """The counter's upper half: elements from 2^34 on (counter 2^32) draw other words than those from 0 on."""
    count = 2 ** 34 + 4096
    x = torch.ones(1, dtype=torch.bfloat16, device="cuda").expand(count // 4096, 4096)  # one value, read at every row
    x = x[:, :1].expand(count // 4096, 4096)
    y = sequence.philox_dropout(torch.ones(1, 4096, dtype=torch.bfloat16, device="cuda").expand(count // 4096, 4096), 0.5, True, 11)
    words = so.philox4x32_10(np.arange(2 ** 32, 2 ** 32 + 1024), 11).reshape(-1)
    assert np.array_equal(_np(y[-1]) != 0, words >= 2 ** 31)
    assert np.array_equal(_np(y[0]) != 0, so.dropout_keep((4096,), 0.5, 11))


# ---- all of them -----------------------------------------------------------------------------------------------------


def test_gradcheck():
    lens = torch.tensor([6, 0, 3], dtype=torch.int32, device="cuda")
    d = dict(device="cuda", dtype=torch.float64)
    x, gate = torch.randn(3, 6, 4, **d).requires_grad_(True), torch.randn(3, 6, 4, **d).requires_grad_(True)
    initial = torch.randn(3, 4, **d).requires_grad_(True)
    for reverse in (False, True):
        assert torch.autograd.gradcheck(lambda a, b, c: sequence.gated_recurrence(a, b, c, lens, reverse), (x, gate, initial))
    packed = torch.randn(2, 20, 6, **d).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda a: sequence.gated_recurrence(a), (packed,))
    w, b = torch.randn(4, **d).requires_grad_(True), torch.randn(4, **d).requires_grad_(True)
    for act in ("none", "silu", "gelu"):
        assert torch.autograd.gradcheck(lambda *a: sequence.group_norm_act(a[0], 2, a[1], a[2], lens, 1e-5, act), (x, w, b))
    assert torch.autograd.gradcheck(lambda a, r: sequence.philox_dropout(a, 0.4, True, 3, r), (x, gate))


def test_no_second_derivative():
    x = torch.randn(2, 4, 6, device="cuda", requires_grad=True)
    for y in (sequence.gated_recurrence(x)[0], sequence.group_norm_act(x, 2), sequence.philox_dropout(x, 0.5)):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once only"):
            g.sum().backward()


def test_no_forward_mode():
    """A tangent on any operand is refused, with and without grad mode, never dropped."""
    import torch.autograd.forward_ad as fwd

    x, row = torch.randn(2, 4, 6, device="cuda"), torch.randn(2, 6, device="cuda")
    calls = [lambda t: sequence.gated_recurrence(t(x))[0], lambda t: sequence.gated_recurrence(x, t(x))[0],
             lambda t: sequence.gated_recurrence(x, x, t(row))[0], lambda t: sequence.group_norm_act(t(x), 2),
             lambda t: sequence.group_norm_act(x, 2, t(row[0])), lambda t: sequence.group_norm_act(x, 2, None, t(row[0])),
             lambda t: sequence.philox_dropout(t(x), 0.5), lambda t: sequence.philox_dropout(x, 0.5, residual=t(x)),
             lambda t: sequence.philox_dropout(x, 0.5, False, residual=t(x)), lambda t: sequence.group_norm_act(t(row), 2)]
    for call in calls:
        for grad_mode in (True, False):
            with fwd.dual_level(), torch.set_grad_enabled(grad_mode), pytest.raises(RuntimeError, match="jvp is not implemented"):
                call(lambda v: fwd.make_dual(v, torch.ones_like(v)))
        call(lambda v: v)  # and nothing is left behind
    for f in (lambda v: sequence.gated_recurrence(v)[0], lambda v: sequence.group_norm_act(v, 2),
              lambda v: sequence.philox_dropout(v, 0.5)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))


def test_refusals():
    x = torch.randn(2, 4, 6, device="cuda")
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="batch, frames, channels"):
        sequence.gated_recurrence(x[0])
    with pytest.raises(RuntimeError, match="even number"):
        sequence.gated_recurrence(x[..., :5])
    with pytest.raises(RuntimeError, match="'gate' to have shape"):
        sequence.gated_recurrence(x, x[..., :5])
    with pytest.raises(RuntimeError, match="same dtype"):
        sequence.gated_recurrence(x, x.half())
    with pytest.raises(RuntimeError, match="'initial' to have shape"):
        sequence.gated_recurrence(x, x, x[:, 0, :3])
    with pytest.raises(RuntimeError, match="must be float16"):
        sequence.gated_recurrence(x.int())
    for bad in (lens.long(), lens.cpu(), lens[:1], lens.view(2, 1)):
        with pytest.raises(RuntimeError, match="lens"):
            sequence.gated_recurrence(x, lens=bad)
        with pytest.raises(RuntimeError, match="lens"):
            sequence.group_norm_act(x, 2, lens=bad)
    with pytest.raises(RuntimeError, match="do not divide"):
        sequence.group_norm_act(x, 4)
    with pytest.raises(RuntimeError, match="do not divide"):
        sequence.group_norm_act(x, 0)
    with pytest.raises(RuntimeError, match="'weight' to have shape"):
        sequence.group_norm_act(x, 2, x[0, 0, :3])
    with pytest.raises(RuntimeError, match="eps"):
        sequence.group_norm_act(x, 2, eps=-1.0)
    with pytest.raises(ValueError, match="activation"):
        sequence.group_norm_act(x, 2, activation="tanh")
    with pytest.raises(RuntimeError, match="lens"):
        sequence.group_norm_act(x.view(2, 2, 2, 6), 2, lens=lens)
    with pytest.raises(ValueError, match="p must be"):
        sequence.philox_dropout(x, -0.1)
    with pytest.raises(RuntimeError, match="same dtype"):
        sequence.philox_dropout(x, 0.1, residual=x.half())
    with pytest.raises(RuntimeError, match="'residual' to have shape"):
        sequence.philox_dropout(x, 0.1, residual=x[:1])
    with pytest.raises(RuntimeError, match="seed tensor"):
        sequence.philox_dropout(x, 0.1, seed=torch.zeros(2, dtype=torch.int64, device="cuda"))
    seed = torch.tensor(3, device="cuda")
    y = sequence.philox_dropout(x.requires_grad_(True), 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_unknown_activation_numbers():
    """The operator's own argument is a 64-bit number: one whose lower half names an activation is none."""
    x = torch.randn(2, 4, 6, device="cuda")
    for act in (4, -1, 2 ** 32, 2 ** 32 + 1):
        with pytest.raises(RuntimeError, match="unknown activation"):
            torch.ops.mellin.group_norm_act(x, 2, act=act)


@pytest.mark.parametrize("frames", [3, 40, 2600])
def test_other_stream_and_captured_graph(frames):
    """The same results on a stream of the caller's, and from a graph that is replayed on other inputs: at a few frames, at
    sizes that one block has, and at sizes that clusters share and whose parameter sums are added by a dependent kernel."""
    lens = torch.tensor([frames, 0, frames * 5 // 8], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(8)
    w, b = (torch.randn(32, device="cuda", generator=gen).requires_grad_(True) for _ in range(2))
    seed = torch.tensor(1, device="cuda")
    x = torch.randn(3, frames, 64, device="cuda", generator=gen)

    def step(x):
        x = x.detach().requires_grad_(True)
        y, final = sequence.gated_recurrence(x, lens=lens)
        z = sequence.group_norm_act(y, 4, w, b, lens, activation="silu")
        out = sequence.philox_dropout(z, 0.2, True, seed, y)
        return [out.detach(), final.detach()] + list(
            torch.autograd.grad([out, final], [x, w, b], [torch.ones_like(out), torch.ones_like(final)]))

    eager = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(eager, other))
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step(static)
    for k in range(3):
        static.copy_(x * (k + 1))
        seed.fill_(k + 1)
        lens.copy_(torch.tensor([frames - k, k, frames // 2], dtype=torch.int32))
        graph.replay()
        want = step(x * (k + 1))
        assert all(torch.equal(a, c) for a, c in zip(captured, want)), k


def test_results_of_two_streams_joined():
    """An operator that takes what another stream's operator writes, after an event: launched dependent on the kernel before
    it in its own stream, it still waits for the other stream, eagerly and in a captured graph."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(8, 3000, 256, device="cuda", generator=gen)
    small = torch.randn(8, 3000, 256, device="cuda", generator=gen)
    side = torch.cuda.Stream()

    def step(x):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            a = x
            for k in range(6):  # long enough to be running still when the other branch is done
                a = sequence.philox_dropout(a, 0.1, True, k)
            a, _ = sequence.gated_recurrence(a, a)
        b = sequence.group_norm_act(small, 4)
        here.wait_stream(side)
        return sequence.philox_dropout(a, 0.2, True, 9, b)

    def in_order(x):
        for k in range(6):
            x = sequence.philox_dropout(x, 0.1, True, k)
        x, _ = sequence.gated_recurrence(x, x)
        torch.cuda.synchronize()
        return sequence.philox_dropout(x, 0.2, True, 9, sequence.group_norm_act(small, 4))

    want = in_order(x)
    for _ in range(5):
        got = step(x)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step(static)
    for k in range(5):
        static.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, in_order(x * (k + 1))), k


def test_entry_points_with_strides_of_the_callers():
    """The C ABI from raw pointers: time running backwards through a negative stride, states off the 16-byte grid."""
    import ctypes

    lib, i64, ptr = capi.lib(), ctypes.c_int64, ctypes.c_void_p
    stream = ptr(torch.cuda.current_stream().cuda_stream)
    for frames in (3, 70, 300):
        n, c = 2, 16
        gen = torch.Generator(device="cuda").manual_seed(frames)
        x, gate, gy = (torch.randn(n, frames, c, device="cuda", generator=gen) for _ in range(3))
        lib.mellin_gated_recurrence_state_count.restype = i64
        count = lib.mellin_gated_recurrence_state_count(i64(n), i64(frames), i64(c))
        y, final = torch.empty_like(x), torch.empty(n, c, device="cuda")
        states = torch.empty(count + 1, device="cuda")[1:]
        last = (frames - 1) * c * 4

        def at(t):
            return [ptr(t.data_ptr() + last), i64(frames * c), i64(-c)]

        assert lib.mellin_gated_recurrence_f32(*at(x), *at(gate), ptr(0), ptr(0), 0, i64(n), i64(frames), i64(c), *at(y),
                                               ptr(final.data_ptr()), ptr(states.data_ptr()), stream) == 0
        xs, gs = x.clone().requires_grad_(True), gate.clone().requires_grad_(True)
        want, want_final = sequence.gated_recurrence(xs, gs, reverse=True)
        want_x, want_g = torch.autograd.grad(want, [xs, gs], gy)
        gx, gg = torch.empty_like(x), torch.empty_like(x)
        assert lib.mellin_gated_recurrence_backward_f32(
            *at(x), *at(gate), ptr(states.data_ptr()), ptr(0), 0, i64(n), i64(frames), i64(c), *at(gy), ptr(0), *at(gx),
            *at(gg), ptr(0), stream) == 0
        # other forms of the same sums: a few units of values of order one to four
        for got, ref in ((y, want), (final, want_final), (gx, want_x), (gg, want_g)):
            assert float((got - ref).detach().abs().max()) <= 1e-5


def test_group_norm_without_epsilon():
    """eps = 0 and an utterance without a frame: nothing of it reaches the parameters' gradients."""
    x = torch.randn(3, 9, 8, device="cuda", requires_grad=True)
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    y = sequence.group_norm_act(x, 2, w, b, torch.tensor([9, 0, 4], dtype=torch.int32, device="cuda"), 0.0, "silu")
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y.sum(), [x, w, b])) and torch.isfinite(y).all()


def test_autocast_meets_in_the_wider_type():
    x = torch.randn(2, 6, 8, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert sequence.philox_dropout(x.bfloat16(), 0.5, True, 1, x).dtype == torch.float32
        assert sequence.gated_recurrence(x.bfloat16(), x)[0].dtype == torch.float32
        assert sequence.group_norm_act(x.bfloat16(), 2).dtype == torch.bfloat16


def test_ordinary_launches_give_the_same():
    """The switch that turns dependent launches off changes no bit."""
    x = torch.randn(3, 2600, 64, device="cuda", requires_grad=True)
    w = torch.randn(64, device="cuda", requires_grad=True)

    def step():
        y, final = sequence.gated_recurrence(x, x)
        z = sequence.philox_dropout(sequence.group_norm_act(y, 2, w, activation="gelu"), 0.3, True, 4, y)
        return [z.detach(), final.detach()] + list(torch.autograd.grad(z.square().sum(), [x, w]))

    first = step()
    before = capi.set_dependent_launch(False)
    try:
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    finally:
        capi.set_dependent_launch(before)


def test_launches():
    """One kernel each way for the recurrence and the dropout."""
    x = torch.randn(2, 40, 64, device="cuda", requires_grad=True)
    before = capi.launch_count()
    y, _ = sequence.gated_recurrence(x)
    assert capi.launch_count() - before == 1
    torch.autograd.grad(y.sum(), x)
    assert capi.launch_count() - before == 2
    z = sequence.philox_dropout(x, 0.5)
    assert capi.launch_count() - before == 3
    torch.autograd.grad(z.sum(), x)
    assert capi.launch_count() - before == 4
    assert capi.device_status() == 0
