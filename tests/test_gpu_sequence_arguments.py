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
