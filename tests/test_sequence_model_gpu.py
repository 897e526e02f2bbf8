"""The sequence operators as they are used together: the residual block, a stream in pieces, the CTC model's step."""
import numpy as np
import pytest
import torch

import ctc_model
import sequence
from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu


def _plain_block(block, x, lens, keep, scale):
    """The block in elementary torch operations (float64), differentiable by autograd; `keep`: the dropout's mask."""
    n, t, c = x.shape
    groups, norm = block.norm.num_groups, block.norm
    rows = []
    for i in range(n):
        length = int(lens[i])
        v = x[i, :length].reshape(length, groups, -1)
        if norm.per_frame:
            d = v - v.mean(2, keepdim=True)
            d = d / (d.square().mean(2, keepdim=True) + norm.eps).sqrt()
        else:
            d = v - v.mean((0, 2), keepdim=True)
            d = d / (d.square().mean((0, 2), keepdim=True) + norm.eps).sqrt()
        z = d.reshape(length, c) * norm.weight + norm.bias
        mix = (z * torch.sigmoid(z)) @ block.recurrence.proj.weight.t() + block.recurrence.proj.bias
        outs, hidden = [], block.recurrence.hidden
        for way in range(block.recurrence.directions):
            value, gate = mix[:, 2 * way * hidden:(2 * way + 1) * hidden], mix[:, (2 * way + 1) * hidden:(2 * way + 2) * hidden]
            h, frames = torch.zeros(hidden, dtype=x.dtype, device=x.device), {}
            for j in (range(length) if way == 0 else reversed(range(length))):
                f = torch.sigmoid(gate[j])
                h = f * h + (1 - f) * value[j]
                frames[j] = h
            outs.append(torch.stack([frames[j] for j in range(length)]))
        y = torch.cat(outs, 1) @ block.out.weight.t() + block.out.bias
        rows.append(x[i, :length] + torch.where(keep[i, :length], y * scale, 0.0))
    return rows


@pytest.mark.parametrize("streaming", [False, True])
def test_block_against_plain_operations(streaming):
    """Values and every gradient in float64.  Both sides are float64 with sums of at most a few thousand terms of order
    one: 2^-53 times a few thousand is 1e-12, and the recurrence adds no more than 1 / (1 - f) ~ 100 of it."""
    torch.manual_seed(7)
    block = sequence.SequenceBlock(24, 20, num_groups=4, dropout=0.3, streaming=streaming).double().cuda()
    with torch.no_grad():
        block.norm.weight.add_(0.3 * torch.randn(24, device="cuda"))
        block.norm.bias.add_(0.3 * torch.randn(24, device="cuda"))
    lens = [40, 1, 23]
    x = torch.randn(3, 40, 24, dtype=torch.float64, device="cuda", requires_grad=True)
    grad = torch.randn(3, 40, 24, dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        grad[i, length:] = 0
    torch.manual_seed(11)
    y, state = block(x, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    params = [x] + list(block.parameters())
    got = torch.autograd.grad(y, params, grad)
    torch.manual_seed(11)
    seed = int(torch.randint(0, 2 ** 62, (1,)).item())
    keep = torch.from_numpy(so.dropout_keep((3, 40, 24), 0.3, seed)).cuda()
    rows = _plain_block(block, x, lens, keep, 1 / 0.7)
    for i, length in enumerate(lens):
        assert float((y[i, :length] - rows[i]).detach().abs().max()) <= 1e-10
    want = torch.autograd.grad(sum((r * grad[i, :len(r)]).sum() for i, r in enumerate(rows)), params)
    for g, w in zip(got, want):
        assert float((g - w).abs().max()) <= 1e-9 * max(1.0, float(w.abs().max()))
    assert state.shape == (1 if streaming else 2, 3, 20)


@pytest.mark.parametrize("streaming", [False, True])
def test_block_with_padding_that_must_not_be_seen(streaming):
    """NaN, infinities and the lowest value behind the utterances' ends, zero gradients there: what is inside them, the
    states and every gradient are those of zero padding."""
    torch.manual_seed(9)
    block = sequence.SequenceBlock(24, 20, num_groups=4, dropout=0.3, streaming=streaming).cuda()
    lens = torch.tensor([40, 0, 23, 45, -2], dtype=torch.int32, device="cuda")
    inside = torch.arange(40, device="cuda")[None, :, None] < lens[:, None, None]
    x = torch.randn(5, 40, 24, device="cuda")
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min], device="cuda").repeat(6)
    grad = torch.where(inside, torch.randn(5, 40, 24, device="cuda"), 0.0)
    results = []
    for padding in (0.0, bad):
        leaf = torch.where(inside, x, padding).requires_grad_(True)
        torch.manual_seed(6)
        y, state = block(leaf, lens)
        grads = torch.autograd.grad(y, [leaf] + list(block.parameters()), grad)
        results.append([torch.where(inside, y, 0.0).detach(), state.detach()] + list(grads))
    for a, b in zip(*results):
        assert torch.isfinite(b).all() and torch.equal(a, b)


def test_per_frame_norm_with_lengths():
    """Frames behind an utterance's end are not read and come out as zeros; lengths that do not fit are refused."""
    norm = sequence.GroupNormAct(3, 12, "gelu", per_frame=True).cuda()
    x = torch.randn(3, 7, 12, device="cuda")
    lens = torch.tensor([7, 0, 4], dtype=torch.int32, device="cuda")
    inside = torch.arange(7, device="cuda")[None, :, None] < lens[:, None, None]
    whole = norm(x)
    y = norm(torch.where(inside, x, float("nan")), lens)
    assert torch.equal(y, torch.where(inside, whole, 0.0))
    time_major = torch.where(inside, x, float("nan")).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(norm(time_major, lens), y)
    assert norm(x[:, :0], lens).shape == (3, 0, 12) and norm(x[:0], lens[:0]).shape == (0, 7, 12)
    for bad in (lens.long(), lens.cpu(), lens[:1], lens.view(3, 1)):
        with pytest.raises(RuntimeError, match="lens"):
            norm(x, bad)
    with pytest.raises(RuntimeError, match="lens"):
        norm(x.view(3, 7, 2, 6).reshape(3, 7, 1, 12), lens)


def test_block_in_a_captured_step():
    """A training step of the block captured with a seed on the device: every replay draws the mask of the seed it finds.
    Without a seed the capture is refused, by the block, the module and the function; in evaluation there is none to draw."""
    torch.manual_seed(4)
    block = sequence.SequenceBlock(32, 16, num_groups=4, dropout=0.4).cuda()
    x, grad = torch.randn(2, 50, 32, device="cuda"), torch.randn(2, 50, 32, device="cuda")
    seed = torch.tensor(3, device="cuda")

    def step(seed):
        leaf = x.detach().requires_grad_(True)
        y, state = block(leaf, seed=seed)
        return [y.detach(), state.detach()] + list(torch.autograd.grad(y, [leaf] + list(block.parameters()), grad))

    side = torch.cuda.Stream()  # warm-up, as captures of library products want it
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(seed)
    masks = []
    for k in (3, 4, 2 ** 62 + 1):
        seed.fill_(k)
        graph.replay()
        want = step(k)
        for got, ref in zip(captured, want):
            # products may be summed in another order under capture: float32 sums of at most 100 terms of order one
            assert float((got - ref).abs().max()) <= 1e-4
        masks.append(captured[0] == x)
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])
    for call in (lambda: block(x), lambda: block.dropout(x), lambda: sequence.philox_dropout(x, 0.4)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="seed"), torch.no_grad(), torch.cuda.graph(graph):
            call()
    block.eval()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        want, _ = block(x)
        with torch.cuda.graph(graph):
            y, _ = block(x)
        graph.replay()
    assert float((y - want).abs().max()) <= 1e-4


def test_stream_in_pieces():
    """A streaming block fed 1, 7, 1, 16, ... frames at a time with its state gives what one call gives, to float32
    rounding: sums over 48 channels and states that forget within ~100 frames, some 1e-5 at values of order one."""
    torch.manual_seed(3)
    block = sequence.SequenceBlock(48, 32, num_groups=6, streaming=True).cuda().eval()
    x = torch.randn(4, 90, 48, device="cuda")
    with torch.no_grad():
        whole, last = block(x)
        state, parts, at = None, [], 0
        for size in [1, 7, 1, 16, 1, 1, 33, 30]:
            y, state = block(x[:, at:at + size], state=state)
            parts.append(y)
            at += size
    assert at == 90
    assert float((torch.cat(parts, 1) - whole).abs().max()) <= 1e-5 and float((state - last).abs().max()) <= 1e-5


def test_block_in_half_precision():
    """bfloat16 parameters and activations, and autocast over float32 parameters: run, finite, near the float32 block."""
    torch.manual_seed(5)
    block = sequence.SequenceBlock(64, num_groups=8, dropout=0.0).cuda()
    x = torch.randn(2, 50, 64, device="cuda")
    lens = torch.tensor([50, 31], dtype=torch.int32, device="cuda")
    want, _ = block(x, lens)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        auto, _ = block(x, lens)
    half, _ = block.bfloat16()(x.bfloat16(), lens)
    # eight roundings to 8 bits of values of order one to four on the way
    for got in (auto, half):
        assert float((got.float() - want)[0].detach().abs().max()) <= 8 * 4 * 2 ** -8
        got.float().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in block.parameters())


def test_ctc_model_with_sequence_blocks():
    """The training step with two blocks runs, its gradients are finite and agree with differences of the loss; what is
    padded on behind an utterance's end changes nothing."""
    torch.manual_seed(1)
    model = ctc_model.MellinCTCNet(channels=(3, 8), bins=11, hidden=32, dropout=0.0, sequence_layers=2,
                                   sequence_groups=4).cuda()
    assert ctc_model.MellinCTCNet(channels=(3, 8), bins=11, hidden=32).state_dict().keys() < model.state_dict().keys()
    x, lens, targets, target_lengths = ctc_model.synthetic_batch([60, 44, 52], 9, "cuda", bins=11)
    targets, target_lengths = targets[:30], torch.tensor([10, 8, 12], device="cuda")

    def loss(x):
        return ctc_model.ctc_loss(model(x, lens), lens, targets, target_lengths)

    value = loss(x)
    value.backward()
    grads = {k: p.grad.clone() for k, p in model.named_parameters()}
    assert all(torch.isfinite(g).all() for g in grads.values())
    longer = torch.nn.functional.pad(x, (0, 8))
    assert abs(float(loss(longer)) - float(value)) <= 1e-5 * abs(float(value))
    # along a random direction of the blocks' parameters: a central difference in float32, step h, is off by about
    # 1e-6 |loss| / h from rounding and h^2 from truncation: 1e-2 relative to a derivative of order one at h = 1e-2
    torch.manual_seed(2)
    names = [k for k in grads if k.startswith("blocks")]
    direction = {k: torch.randn_like(grads[k]) / len(names) for k in names}
    slope = sum(float((grads[k] * direction[k]).sum()) for k in names)
    values = []
    for step in (1e-2, -1e-2):
        with torch.no_grad():
            for k, p in model.named_parameters():
                if k in direction:
                    p.add_(step * direction[k])
            values.append(float(loss(x)))
            for k, p in model.named_parameters():
                if k in direction:
                    p.sub_(step * direction[k])
    assert abs((values[0] - values[1]) / 2e-2 - slope) <= 2e-2 * max(1.0, abs(slope))
    step = ctc_model.TrainStep(model)
    assert np.isfinite(float(step(x, lens, targets, target_lengths)))
