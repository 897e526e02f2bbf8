"""Sequence operators on per-frame features: what carries information over an utterance's frames.

The reference's acoustic model runs a recurrent layer between its convolutions and its output (``models.py:435-445``;
torch's RNN / LSTM / GRU there) with dropout around it.  Here that place is taken by three operators on (batch, frames,
channels) tensors, channels last, each a hand-written CUDA kernel forward and backward:

* :func:`gated_recurrence`: a linear recurrence whose gates depend on the frame, a scan over the frames of ragged
  utterances (``csrc/recurrence.cu``);
* :func:`group_norm_act`: group norm over an utterance's frames with an activation (``csrc/group_norm.cu``);
* :func:`philox_dropout`: dropout whose mask comes from a counter-based generator and is never stored, with an optional
  residual (``csrc/philox_dropout.cu``);

and by :class:`SequenceBlock`, which runs them as one residual block.  float16, bfloat16, float32 and float64 tensors;
sums, states and statistics are float32 (float64 for float64).  There is no CPU path: the operators raise on tensors
that are not on a CUDA device.
"""
from typing import Optional, Tuple, Union

import torch

import mconv  # noqa: F401  (loads the extension that registers torch.ops.mellin.*)

__all__ = ["gated_recurrence", "group_norm_act", "philox_dropout", "GatedRecurrence", "GroupNormAct", "PhiloxDropout",
           "SequenceBlock"]

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _on_device(c: str, x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError("%s: expected a CUDA tensor (there is no CPU implementation)" % c)


def gated_recurrence(
    input: torch.Tensor,
    gate: Optional[torch.Tensor] = None,
    initial: Optional[torch.Tensor] = None,
    lens: Optional[torch.Tensor] = None,
    reverse: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""``h_t = f_t h_{t-1} + (1 - f_t) x_t`` with ``f = sigmoid(gate)``; returns ``(output, final)``.

    ``input`` and ``gate`` are (batch, frames, channels); without ``gate``, ``input`` is (batch, frames, 2 channels) and
    holds the values in its first half and the gates in its second (one projection, no copies, one gradient).  Strides
    between utterances and frames are free: a time-major tensor is passed as ``x.transpose(0, 1)`` and gets a time-major
    output.  ``lens`` (int32 CUDA tensor, one length per utterance): frames behind an utterance's end are never read,
    their outputs and gradients are zero.  ``reverse``: from an utterance's last frame to its first.  ``initial``
    (batch, channels) is the state before the first frame met, zeros when not given; ``final`` the state after the last
    one met, float32 (float64 for float64 input) whatever the input's type, so that a stream fed in pieces, down to one
    frame a call, carries it unrounded.  The frames are joined in runs, so an infinite value makes those after it infinite
    or NaN.  Differentiable in input, gate and initial."""
    _on_device("gated_recurrence", input)
    return torch.ops.mellin.gated_recurrence(input, gate, initial, lens, reverse)


def group_norm_act(
    input: torch.Tensor,
    num_groups: int,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    lens: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    activation: str = "relu",
) -> torch.Tensor:
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` on (batch, ..., channels), channels last.

    Mean and biased variance of an utterance's group of ``channels / num_groups`` adjacent channels over everything
    between the first and the last dimension, or, with ``lens`` and a (batch, frames, channels) input, over the
    utterance's own frames: those behind its end are never read, their outputs and gradients are zero.  ``activation``:
    ``"none"``, ``"relu"``, ``"silu"`` or ``"gelu"`` (with the error function).  Differentiable in input, weight and bias;
    the parameters' gradients are summed in a fixed order.  ReLU's slope is that of the side on which its argument falls as
    computed in float32; where 64 bits have the argument within about 2e-8 of zero that may be the other side (one of 16
    million elements, in one call of ten), and a parameter's gradient then differs by that element's whole term.
    A group whose squared deviations pass the statistics' type (float32 ends at 3.4e38) has no finite variance and comes out
    as NaN or ``act(bias)``.  Batch times channels is below 2^31."""
    _on_device("group_norm_act", input)
    if activation not in ACTIVATIONS:
        raise ValueError("group_norm_act: activation must be one of %s, got %r" % (sorted(ACTIVATIONS), activation))
    return torch.ops.mellin.group_norm_act(input, num_groups, weight, bias, lens, eps, ACTIVATIONS[activation])


def philox_dropout(
    input: torch.Tensor,
    p: float = 0.5,
    training: bool = True,
    seed: Union[None, int, torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Dropout, plus ``residual`` when given; the mask is a function of ``seed`` and of an element's offset.

    Element ``i`` (row-major offset) is dropped where word ``i % 4`` of Philox4x32-10 at counter ``i // 4`` with key
    ``seed`` is below ``floor(p * 2**32 + 0.5)``; the others are scaled by ``1 / (1 - p)``.  The mask is never stored:
    backward draws it again.  A dropped element is zero whatever ``input`` holds there.  ``seed``: an integer of 64 bits, or an int64
    CUDA tensor of one element that is read when the kernel runs (so that a captured graph draws a new mask at each
    replay after the tensor is overwritten); drawn from torch's default CPU generator when not given, so
    ``torch.manual_seed`` governs it (refused while a graph is captured: every replay would draw the one mask).  In evaluation
    nothing is dropped.  Differentiable in input and residual."""
    _on_device("philox_dropout", input)
    if not 0.0 <= p <= 1.0:
        raise ValueError("philox_dropout: p must be in [0, 1], got %r" % (p,))
    if not training or p == 0.0:
        return input if residual is None else torch.ops.mellin.philox_dropout(input, 0.0, 0, None, residual)
    if isinstance(seed, torch.Tensor):
        return torch.ops.mellin.philox_dropout(input, p, 0, seed, residual)
    if seed is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("philox_dropout: a seed drawn while a graph is captured would be every replay's: pass `seed`, "
                               "a CUDA tensor that is overwritten between replays (or an int, to keep one mask)")
        seed = int(torch.randint(0, 2 ** 62, (1,), device="cpu").item())
    else:
        seed = int(seed) & ((1 << 64) - 1)
    return torch.ops.mellin.philox_dropout(input, p, seed - (1 << 64) if seed >> 63 else seed, None, residual)


class GatedRecurrence(torch.nn.Module):
    """A projection to values and gates, then :func:`gated_recurrence`, one way or both ways.

    ``forward(x, lens=None, state=None)`` with ``x`` (batch, frames, in_features) returns ``(output, state)``: the output
    (batch, frames, hidden * directions) and the final states (directions, batch, hidden), which the next call takes when
    a stream comes in pieces (one way only: the other direction needs the end first)."""

    def __init__(self, in_features: int, hidden: int, bidirectional: bool = False):
        super().__init__()
        self.hidden, self.bidirectional = hidden, bidirectional
        self.directions = 2 if bidirectional else 1
        self.proj = torch.nn.Linear(in_features, 2 * hidden * self.directions)
        self.reset_parameters()

    def extra_repr(self) -> str:
        return f"hidden={self.hidden}, bidirectional={self.bidirectional}"

    def reset_parameters(self) -> None:
        self.proj.reset_parameters()
        with torch.no_grad():  # gates that start out remembering: sigmoid(1) = 0.73 of the state is kept
            for way in range(self.directions):
                self.proj.bias[(2 * way + 1) * self.hidden:(2 * way + 2) * self.hidden].add_(1.0)

    def forward(self, x: torch.Tensor, lens: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None):
        if state is not None and self.bidirectional:
            raise RuntimeError("GatedRecurrence: a two-way layer cannot go on from a state")
        mix = self.proj(x)
        if not self.bidirectional:
            y, final = gated_recurrence(mix, None, None if state is None else state[0], lens)
            return y, final.unsqueeze(0)
        ahead, back = mix.split(2 * self.hidden, dim=2)
        y0, f0 = gated_recurrence(ahead, lens=lens)
        y1, f1 = gated_recurrence(back, lens=lens, reverse=True)
        return torch.cat((y0, y1), 2), torch.stack((f0, f1))


def _present(x: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
    """1 for each of x's frames, one after the other, that is inside its utterance, else 0."""
    if x.dim() != 3:
        raise RuntimeError("GroupNormAct: 'lens' goes with a (batch, frames, channels) input")
    if not lens.is_cuda or lens.dtype != torch.int32 or lens.shape != x.shape[:1] or lens.device != x.device:
        raise RuntimeError("GroupNormAct: 'lens' must be an int32 CUDA tensor on the input's device with one length per utterance")
    return (torch.arange(x.shape[1], dtype=torch.int32, device=x.device) < lens[:, None]).int().reshape(-1)


class GroupNormAct(torch.nn.Module):
    """:func:`group_norm_act` with learnable ``weight`` and ``bias`` (names and shapes of ``torch.nn.GroupNorm``).

    ``per_frame``: the statistics of each frame by itself, as a stream that comes in pieces needs them (the frames are then
    the batch: utterances times frames times channels is below 2^31).  ``lens`` as in :func:`group_norm_act` either way."""

    def __init__(self, num_groups: int, num_channels: int, activation: str = "relu", eps: float = 1e-5,
                 per_frame: bool = False):
        super().__init__()
        if num_channels % num_groups:
            raise ValueError("GroupNormAct: num_channels must be divisible by num_groups")
        if activation not in ACTIVATIONS:
            raise ValueError("GroupNormAct: activation must be one of %s, got %r" % (sorted(ACTIVATIONS), activation))
        self.num_groups, self.activation, self.eps, self.per_frame = num_groups, activation, eps, per_frame
        self.weight = torch.nn.Parameter(torch.ones(num_channels))
        self.bias = torch.nn.Parameter(torch.zeros(num_channels))

    def extra_repr(self) -> str:
        return (f"{self.num_groups}, {self.weight.numel()}, activation={self.activation}, eps={self.eps}, "
                f"per_frame={self.per_frame}")

    def forward(self, x: torch.Tensor, lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.per_frame:
            rows = x.reshape(-1, 1, x.shape[-1])  # every frame an utterance of its own, which is there (1) or not (0)
            y = group_norm_act(rows, self.num_groups, self.weight, self.bias, None if lens is None else _present(x, lens),
                               self.eps, self.activation)
            return y.view(x.shape)
        return group_norm_act(x, self.num_groups, self.weight, self.bias, lens, self.eps, self.activation)


class PhiloxDropout(torch.nn.Module):
    """:func:`philox_dropout` as a module: ``forward(x, residual=None)``."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("PhiloxDropout: p must be in [0, 1], got %r" % (p,))
        self.p = p

    def extra_repr(self) -> str:
        return f"p={self.p}"

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                seed: Union[None, int, torch.Tensor] = None) -> torch.Tensor:
        return philox_dropout(x, self.p, self.training, seed, residual)


class SequenceBlock(torch.nn.Module):
    """``x + dropout(out(recurrence(norm_act(x))))`` on (batch, frames, channels).

    ``forward(x, lens=None, state=None, seed=None)`` returns ``(output, state)``.  ``streaming``: one way and the norm frame
    by frame, so that feeding a stream in pieces with the state passed on gives what one call over all of it gives; otherwise the
    recurrence runs both ways and the norm's statistics are an utterance's.  Frames behind an utterance's end come out
    as they went in plus the output layer's bias: finite where ``x`` is, and never read by the next block.  ``seed``: the
    dropout's, as :func:`philox_dropout` takes it; a captured training step needs it, one for each block (blocks of one shape
    that share a seed drop the same elements)."""

    def __init__(self, channels: int, hidden: Optional[int] = None, num_groups: int = 32, activation: str = "silu",
                 dropout: float = 0.05, streaming: bool = False):
        super().__init__()
        hidden = channels if hidden is None else hidden
        self.norm = GroupNormAct(num_groups, channels, activation, per_frame=streaming)
        self.recurrence = GatedRecurrence(channels, hidden, bidirectional=not streaming)
        self.out = torch.nn.Linear(hidden * self.recurrence.directions, channels)
        self.dropout = PhiloxDropout(dropout)

    def forward(self, x: torch.Tensor, lens: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                seed: Union[None, int, torch.Tensor] = None):
        y, state = self.recurrence(self.norm(x, lens), lens, state)
        return self.dropout(self.out(y), x, seed), state
