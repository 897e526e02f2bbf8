"""The sequence operators where no GPU is needed: the generator against its published vectors, the oracle against
differences, the argument checks of the C entry points and of the Python surface."""
import ctypes

import numpy as np
import pytest
import torch

import capi
import sequence
from oracle import sequence_oracle as so

I64, NULL = ctypes.c_int64, ctypes.c_void_p(0)
BAD, WORKSPACE, UNSUPPORTED = 1, 3, 4


def test_philox_vectors():
    """Known-answer vector of the generator's authors: counter 0, key 0."""
    words = so.philox4x32_10([0], 0)[0]
    assert [int(w) for w in words] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_keep_rate_of_the_oracle():
    for p in (0.05, 0.5, 0.9):
        count = 1 << 16
        kept = so.dropout_keep((count,), p, 0x1234567890ABCDEF).mean()
        assert abs(kept - (1 - p)) <= 5 * (p * (1 - p) / count) ** 0.5
    assert so.dropout_keep((1000,), 0.0, 3).all() and not so.dropout_keep((1000,), 1.0, 3).any()


@pytest.mark.parametrize("reverse", [False, True])
def test_oracle_recurrence_gradients_against_differences(reverse):
    rng = np.random.default_rng(3)
    n, t, c, lens = 3, 7, 2, [7, 0, 4]
    args = {"x": rng.standard_normal((n, t, c)), "gate": rng.standard_normal((n, t, c)),
            "initial": rng.standard_normal((n, c))}
    gy, gf = rng.standard_normal((n, t, c)), rng.standard_normal((n, c))

    def loss(**a):
        r = so.recurrence(lens=lens, reverse=reverse, **a)
        return (r["y"][0] * gy).sum() + (r["final"][0] * gf).sum()

    grads = so.recurrence(lens=lens, reverse=reverse, grad_y=gy, grad_final=gf, **args)
    for name, got in (("x", grads["grad_x"][0]), ("gate", grads["grad_gate"][0]), ("initial", grads["grad_initial"][0])):
        for at in np.ndindex(args[name].shape):
            up, down = {k: v.copy() for k, v in args.items()}, {k: v.copy() for k, v in args.items()}
            up[name][at] += 1e-5
            down[name][at] -= 1e-5
            # central difference: truncation step^2 ~ 1e-10, rounding 1e-16 * |loss| / step ~ 1e-10
            assert abs((loss(**up) - loss(**down)) / 2e-5 - got[at]) <= 1e-8


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_oracle_norm_gradients_against_differences(act):
    rng = np.random.default_rng(4)
    n, t, c, lens = 3, 4, 6, [4, 0, 2]
    args = {"x": rng.standard_normal((n, t, c)), "weight": rng.standard_normal(c), "bias": rng.standard_normal(c)}
    gy = rng.standard_normal((n, t, c))

    def loss(**a):
        return (so.group_norm_act(groups=3, lens=lens, act=act, **a)["y"][0] * gy).sum()

    grads = so.group_norm_act(groups=3, lens=lens, act=act, grad_y=gy, **args)
    for name in args:
        for at in np.ndindex(args[name].shape):
            up, down = {k: v.copy() for k, v in args.items()}, {k: v.copy() for k, v in args.items()}
            up[name][at] += 1e-5
            down[name][at] -= 1e-5
            assert abs((loss(**up) - loss(**down)) / 2e-5 - grads["grad_" + name][0][at]) <= 1e-7


def _recurrence(lib, sfx, batch, frames, channels):
    return getattr(lib, "mellin_gated_recurrence" + sfx)(
        NULL, I64(0), I64(0), NULL, I64(0), I64(0), NULL, NULL, 0, I64(batch), I64(frames), I64(channels), NULL, I64(0),
        I64(0), NULL, NULL, NULL)


@pytest.mark.parametrize("sfx", ["_f32", "_f64", "_f16", "_bf16"])
def test_entry_points_validate_before_touching_the_device(sfx):
    lib = capi.lib()
    assert _recurrence(lib, sfx, -1, 4, 4) == BAD and b"negative extent" in lib.mellin_last_error()
    assert _recurrence(lib, sfx, 2, 4, 4) == BAD and b"null pointer" in lib.mellin_last_error()
    assert _recurrence(lib, sfx, 2 ** 31, 4, 4) == UNSUPPORTED
    assert _recurrence(lib, sfx, 0, 4, 4) == 0 and _recurrence(lib, sfx, 2, 4, 0) == 0
    back = getattr(lib, "mellin_gated_recurrence_backward" + sfx)
    assert back(NULL, I64(0), I64(0), NULL, I64(0), I64(0), NULL, NULL, 0, I64(2), I64(4), I64(4), NULL, I64(0), I64(0),
                NULL, NULL, I64(0), I64(0), NULL, I64(0), I64(0), NULL, NULL) == BAD
    norm = getattr(lib, "mellin_group_norm_act" + sfx)

    def call(batch, frames, channels, groups, act=0, ws=NULL, nbytes=0):
        return norm(NULL, I64(0), I64(0), NULL, NULL, NULL, I64(batch), I64(frames), I64(channels), I64(groups),
                    ctypes.c_double(1e-5), act, NULL, I64(0), I64(0), NULL, ws, ctypes.c_size_t(nbytes), NULL)

    assert call(2, 4, 6, 4) == BAD and b"groups" in lib.mellin_last_error()
    assert call(2, 4, 6, 0) == BAD and call(2, 4, 6, 3, act=7) == BAD
    assert call(0, 4, 6, 3) == 0
    size = getattr(lib, "mellin_group_norm_act_workspace_bytes" + sfx)
    assert size(2, 4, 6, 3, 0) == 0 and call(2, 4, 6, 3) == BAD and b"null pointer" in lib.mellin_last_error()
    assert size(1, 9000, 8192, 1, 0) > 0 and call(1, 9000, 8192, 1) == WORKSPACE and b"workspace" in lib.mellin_last_error()
    assert size(-1, 4, 6, 3, 1) == 0 and size(2, 4, 6, 4, 1) == 0
    drop = getattr(lib, "mellin_philox_dropout" + sfx)

    def dropout(rows, cols, p):
        return drop(NULL, I64(cols), NULL, I64(0), I64(rows), I64(cols), ctypes.c_double(p), ctypes.c_uint64(1), NULL, NULL,
                    NULL)

    assert dropout(1, -1, 0.5) == BAD and dropout(1, 8, 1.5) == BAD and dropout(1, 8, float("nan")) == BAD
    assert dropout(1, 8, 0.5) == BAD and b"null pointer" in lib.mellin_last_error()
    assert dropout(1, 0, 0.5) == 0


def test_state_count():
    count = capi.lib().mellin_gated_recurrence_state_count
    count.restype = I64
    assert count(I64(2), I64(0), I64(5)) == 0 and count(I64(2), I64(1), I64(5)) == 10
    assert count(I64(2), I64(-1), I64(5)) == 0 and count(I64(3), I64(1000), I64(7)) >= 3 * 7


def test_python_surface_refuses():
    x = torch.zeros(2, 3, 4)
    for call in (lambda: sequence.gated_recurrence(x), lambda: sequence.group_norm_act(x, 2),
                 lambda: sequence.philox_dropout(x, 0.5)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="divisible"):
        sequence.GroupNormAct(3, 4)
    with pytest.raises(ValueError, match="activation"):
        sequence.GroupNormAct(2, 4, activation="tanh")
    with pytest.raises(ValueError, match="p must be"):
        sequence.PhiloxDropout(1.5)
    with pytest.raises(RuntimeError, match="two-way"):
        sequence.GatedRecurrence(4, 4, bidirectional=True)(x, state=torch.zeros(2, 2, 4))


def test_block_parameters():
    block = sequence.SequenceBlock(64, 32, num_groups=4)
    assert {k: tuple(v.shape) for k, v in block.state_dict().items()} == {
        "norm.weight": (64,), "norm.bias": (64,), "recurrence.proj.weight": (128, 64), "recurrence.proj.bias": (128,),
        "out.weight": (64, 64), "out.bias": (64,)}
    one_way = sequence.SequenceBlock(64, 32, num_groups=4, streaming=True)
    assert one_way.recurrence.directions == 1 and one_way.norm.per_frame
    assert "hidden=32" in repr(block) and "p=0.05" in repr(block)


def test_statistics_offsets_beyond_32_bits(tmp_path):
    """The kernels' offset into (batch, groups, 2) statistics, compiled for the host, at the largest extents that the entry
    points admit (batch * groups below 2^31): no launch of that size is needed to see it wrap."""
    import os
    import re
    import subprocess

    csrc = os.path.join(os.path.dirname(os.path.abspath(capi.__file__)), "csrc")
    source = tmp_path / "offset.cpp"
    source.write_text('#include "sequence_index.h"\n'
                      'extern "C" long long offset(int n, int groups, int g) { return mellin::seq::stats_offset(n, groups, g); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", csrc, str(source), "-o", str(tmp_path / "offset.so")],
                   check=True)
    offset = ctypes.CDLL(str(tmp_path / "offset.so")).offset
    offset.restype, offset.argtypes = ctypes.c_longlong, [ctypes.c_int] * 3
    for batch, groups in ((1, 1), (3, 32), (2 ** 20, 1024), (2 ** 21 - 1, 1024), (1, 2 ** 30), (2 ** 31 - 1, 1), (46340, 46341)):
        for n, g in ((0, 0), (batch - 1, 0), (batch - 1, groups - 1), (batch // 2, groups // 2)):
            assert offset(n, groups, g) == (n * groups + g) * 2
    # and every access to the statistics in the kernels goes through it
    text = open(os.path.join(csrc, "group_norm.cu")).read()
    uses = re.findall(r"a\.stats(?:_out)? \+ (\w+)|a\.stats(?:_out)?(\[)", text)
    assert len(uses) == 5 and all(use == ("stats_offset", "") for use in uses)


@pytest.mark.parametrize("sfx", ["_f32", "_f64", "_f16", "_bf16"])
def test_recurrence_refuses_what_no_device_holds(sfx):
    """256 frames that lie 2^31 elements apart: refused before anything is launched (the pointers are no memory)."""
    lib, at, far = capi.lib(), ctypes.c_void_p(4096), 2 ** 31
    dense = [at, I64(300 * 8), I64(8)]
    for forward in ([at, I64(0), I64(far)] + dense + [NULL, NULL, 0, I64(1), I64(300), I64(8)] + dense,
                    dense + [at, I64(0), I64(far)] + [NULL, NULL, 1, I64(1), I64(300), I64(8)] + dense,
                    dense + dense + [NULL, NULL, 0, I64(1), I64(300), I64(8)] + [at, I64(0), I64(far)]):
        assert getattr(lib, "mellin_gated_recurrence" + sfx)(*forward, NULL, NULL, NULL) == UNSUPPORTED
        assert b"between them" in lib.mellin_last_error()
    back = getattr(lib, "mellin_gated_recurrence_backward" + sfx)
    assert back(*dense, *dense, at, NULL, 0, I64(1), I64(300), I64(8), at, I64(0), I64(far), NULL, *dense, *dense, NULL,
                NULL) == UNSUPPORTED


@pytest.mark.parametrize("sfx", ["_f32", "_f64", "_f16", "_bf16"])
def test_norm_refuses_a_bad_epsilon(sfx):
    lib = capi.lib()
    for eps in (-1e-5, float("nan"), float("-inf")):
        assert getattr(lib, "mellin_group_norm_act" + sfx)(
            NULL, I64(0), I64(0), NULL, NULL, NULL, I64(0), I64(4), I64(6), I64(3), ctypes.c_double(eps), 0, NULL, I64(0),
            I64(0), NULL, NULL, ctypes.c_size_t(0), NULL) == BAD
        assert b"eps" in lib.mellin_last_error()
