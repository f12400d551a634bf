"""Operands of the sequence operators that are refused on the GPU, and what its calls leave behind."""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import ops

pytestmark = pytest.mark.gpu


def test_int4_scale_of_a_single_row():
    """One row in 8 bits with the scale of no dimensions that the norm gives it; a scale elsewhere is refused."""
    gen = torch.Generator().manual_seed(1)
    packed = torch.randint(0, 256, (7, 32), generator=gen, dtype=torch.uint8).cuda()
    scales = torch.rand(7, 2, generator=gen).cuda()
    q, scale = ops.rms_norm(torch.randn(64, generator=gen).cuda(), quantize="int8")
    assert scale.shape == ()
    y = ops.int4_linear(q, packed, scales, x_scale=scale)
    assert torch.equal(y, ops.int4_linear(q[None], packed, scales, x_scale=scale[None])[0])
    with pytest.raises(ValueError, match="device"):
        ops.int4_linear(q, packed, scales, x_scale=scale.cpu())
    with pytest.raises(NotImplementedError, match="x_scale"):
        ops.int4_linear(q, packed, scales, x_scale=scale.double())


def test_a_state_stepped_after_it_was_saved_has_no_gradient():
    """Torch's own error in place of gradients at another state."""
    gen = torch.Generator().manual_seed(2)
    x, delta, b, c = (torch.randn(2, 5, n, generator=gen).cuda() for n in (16, 16, 4, 4))
    a, state = -torch.rand(16, 4, generator=gen).cuda(), torch.randn(2, 16, 4, generator=gen).cuda()
    leaf = x.clone().requires_grad_()
    y = ops.selective_scan(leaf, delta, a, b, c, softplus=True, state=state)
    ops.selective_scan_step(state, x[:, 0], delta[:, 0], a, b[:, 0], c[:, 0], softplus=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    taps, weight = torch.randn(2, 3, 16, generator=gen).cuda(), torch.randn(16, 4, generator=gen).cuda()
    y = ops.causal_conv1d(leaf, weight, state=taps)
    ops.causal_conv1d_step(taps, x[:, 0], weight)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_of_no_tokens():
    """Of a length of zero the state's gradient comes back as it is, and the parameters' are zero."""
    gen = torch.Generator().manual_seed(3)
    x, bc = torch.zeros(2, 0, 8).cuda(), torch.zeros(2, 0, 4).cuda()
    a, state, seed = (torch.randn(*s, generator=gen).cuda().requires_grad_() for s in ((8, 4), (2, 8, 4), (2, 8, 4)))
    _, last = ops.selective_scan(x, x, a, bc, bc, state=state, return_state=True)
    da, dstate = torch.autograd.grad(last, [a, state], seed.detach())
    assert not da.any() and torch.equal(dstate, seed)
    weight, taps, seed = (torch.randn(*s, generator=gen).cuda().requires_grad_() for s in ((8, 4), (2, 3, 8), (2, 3, 8)))
    _, new = ops.causal_conv1d(x, weight, state=taps, return_state=True)
    dweight, dtaps = torch.autograd.grad(new, [weight, taps], seed.detach())
    assert not dweight.any() and torch.equal(dtaps, seed)


def test_a_prompt_of_more_tokens_than_a_grid_holds():
    """17 sequences of 4000 tokens through the quantised stack; the first of them alone gives the same logits (within the
    few flips of 8-bit codes that test_gpu_state_space.py allows for)."""
    from extended_einsum_b200.state_space import SelectiveStack, StackShape, init_parameters

    shape = StackShape(layers=1, width=64, channels=64, states=4, outputs=32)
    model = SelectiveStack(shape, init_parameters(shape, torch.Generator().manual_seed(4)), torch.float32).quantize()
    tokens = torch.randint(shape.outputs, (17, 4000), generator=torch.Generator().manual_seed(5)).cuda()
    logits = model.prompt(tokens, model.empty_state(17))
    alone = model.prompt(tokens[:1], model.empty_state(1))
    assert logits.shape == (17, 4000, 32) and torch.isfinite(logits).all()
    torch.testing.assert_close(logits[:1].float(), alone.float(), rtol=0.05, atol=0.05 * alone.abs().max().item())
