"""The state space stack: a training step lowers the loss, and prompts and single tokens agree."""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import ops
from extended_einsum_b200.state_space import QuantizedStack, SelectiveStack, StackShape, init_parameters

pytestmark = pytest.mark.gpu

SHAPE = StackShape(layers=2, width=96, channels=160, states=8, outputs=64)


def stack(dtype):
    return SelectiveStack(SHAPE, init_parameters(SHAPE, torch.Generator().manual_seed(0)), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_learns_a_repeating_sequence(dtype):
    model = stack(dtype)
    tensors = [t.requires_grad_() for t in model.tensors()]
    tokens = torch.arange(7).repeat(2, 9)[:, :60].cuda()
    optimizer = torch.optim.Adam(tensors, lr=3e-3)
    losses = []
    for _ in range(30):
        logits = model.forward(tokens[:, :-1]).float()
        loss = torch.nn.functional.cross_entropy(logits.reshape(-1, SHAPE.outputs), tokens[:, 1:].reshape(-1))
        optimizer.zero_grad()
        loss.backward()
        assert all(t.grad is not None and torch.isfinite(t.grad).all() for t in tensors)
        optimizer.step()
        losses.append(loss.item())
    assert losses[-1] < 0.5 * losses[0], losses


def test_prompts_and_single_tokens_agree():
    """Float32 activations: a ragged prompt followed by single tokens gives the logits of the whole sequences.  The norm's
    8-bit codes of a value at a rounding boundary may fall either way, one step of 1/16 of the value: a few such
    flips among 96 inputs move the logits by a few hundredths of their size."""
    model: QuantizedStack = stack(torch.float32).quantize()
    gen = torch.Generator().manual_seed(1)
    tokens = torch.randint(SHAPE.outputs, (3, 40), generator=gen).cuda()
    lengths = torch.tensor([25, 1, 17])
    whole = model.prompt(tokens, model.empty_state(3))
    state = model.empty_state(3)
    part = model.prompt(tokens[:, :25], state, lengths.cuda())
    for i, n in enumerate(lengths.tolist()):
        torch.testing.assert_close(part[i, :n], whole[i, :n], rtol=0.05, atol=0.05 * whole.abs().max().item())
    for k in range(10):
        at = lengths + k
        logits = model.step(tokens[torch.arange(3), at.cuda()], state)
        want = whole[torch.arange(3), at.cuda()]
        torch.testing.assert_close(logits, want, rtol=0.05, atol=0.05 * whole.abs().max().item())


def test_gpu_operands_that_do_not_fit_are_refused():
    x = torch.zeros(2, 5, 16, device="cuda")
    one = torch.zeros(16, 4, device="cuda")
    bc = torch.zeros(2, 5, 4, device="cuda")
    with pytest.raises(ValueError, match="shape"):
        ops.selective_scan(x, x[:, :4], one, bc, bc)
    with pytest.raises(NotImplementedError, match="delta"):
        ops.selective_scan(x, x.bfloat16(), one, bc, bc)
    with pytest.raises(ValueError, match="groups"):
        ops.selective_scan(x, x, one, torch.zeros(2, 5, 3, 4, device="cuda"), torch.zeros(2, 5, 3, 4, device="cuda"))
    with pytest.raises(NotImplementedError, match="64"):
        wide = torch.zeros(2, 5, 65, device="cuda")
        ops.selective_scan(x, x, torch.zeros(16, 65, device="cuda"), wide, wide)
    with pytest.raises(ValueError, match="device"):
        ops.selective_scan(x, x, one.cpu(), bc, bc)
    with pytest.raises(NotImplementedError, match="float64"):
        ops.rms_norm(x.double())
    with pytest.raises(ValueError, match="quantize"):
        ops.rms_norm(x, quantize="int4")
    with pytest.raises(NotImplementedError, match="backward"):
        ops.rms_norm(x.clone().requires_grad_(), quantize="e4m3")
    with pytest.raises(ValueError, match="activation"):
        ops.causal_conv1d(x, one, activation="gelu")
    with pytest.raises(NotImplementedError, match="width"):
        ops.causal_conv1d(x, torch.zeros(16, 5, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        ops.causal_conv1d_step(torch.zeros(2, 16, 3, device="cuda").transpose(1, 2), x[:, 0], one)
    with pytest.raises(NotImplementedError, match="backward"):
        ops.selective_scan_step(torch.zeros(2, 16, 4, device="cuda"), x[:, 0].clone().requires_grad_(), x[:, 0], one, bc[:, 0], bc[:, 0])
    packed = torch.zeros(3, 8, dtype=torch.uint8, device="cuda")
    with pytest.raises(NotImplementedError, match="multiple of 32"):
        ops.int4_linear(x, packed, torch.zeros(3, 1, device="cuda"))
    with pytest.raises(ValueError, match="x_scale"):
        ops.int4_linear(x, packed, torch.zeros(3, 1, device="cuda"), x_scale=torch.zeros(2, 5, device="cuda"))
