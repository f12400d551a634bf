"""Values that are not finite, at places where they must not spread (the scan's masked positions)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_sequence import close, cuda, leaf, randn, scan_call, scan_inputs, scan_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length,channels", [(50, 40), (700, 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_gradients_past_the_end_are_zero_whatever_comes_back(dtype, length, channels):
    """A gradient of the last state that has overflowed, and a state that has: the positions past a sequence's end still have
    zero gradients, a sequence of no tokens hands the gradient on, and the other sequences do not notice."""
    ends = [0, 21, length, 5]
    v = scan_inputs(61, 4, length, channels, 16, 1, dtype)
    names = list(v)
    gen = torch.Generator().manual_seed(62)
    dy, dstate = randn(gen, 4, length, channels, dtype=dtype).cuda(), randn(gen, 4, channels, 16).cuda()
    lengths = torch.tensor(ends).cuda()

    def gradients(inputs, seed):
        g = leaf({k: cuda(t) for k, t in inputs.items()}, names)
        out = scan_call(g, True, lengths, return_state=True)
        return dict(zip(names, torch.autograd.grad(out, [g[k] for k in names], [dy, seed])))

    clean = gradients(v, dstate)
    spoilt = dstate.clone()
    spoilt[0] = float("inf")
    got = gradients(v, spoilt)
    assert torch.equal(got["state"][0], spoilt[0])
    for k in names:
        if k == "state":
            assert torch.equal(got[k][1:], clean[k][1:])
        else:
            assert torch.equal(got[k], clean[k]), k
    spoilt[1] = float("inf")
    v["state"][3] = float("inf")
    got = gradients(v, spoilt)
    for k in ("x", "delta", "b", "c", "z"):
        for i, end in enumerate(ends):
            assert not got[k][i, end:].any(), (k, i)
        assert torch.equal(got[k][2], clean[k][2])


@pytest.mark.parametrize("length,channels,ends", [(1, 24, None), (37, 40, None), (60, 24, [0, 5, 60]), (700, 24, [700, 0, 130])])
def test_scan_rates_of_minus_infinity(length, channels, ends):
    """A state that does not outlast a token (a = -exp(a large number)): beyond a sequence's end, and in the rest of a
    tile, no token passes and the state stays."""
    batch = 1 if ends is None else 3
    v = scan_inputs(63 + length, batch, length, channels, 16)
    v["a"][::2, 3], v["a"][1, :], v["a"][2, 5] = float("-inf"), float("-inf"), -3e38
    lengths = None if ends is None else torch.tensor(ends).cuda()
    g = leaf({k: cuda(t) for k, t in v.items()}, ["x", "delta"])
    y, state = scan_call(g, True, lengths, return_state=True)
    want_y, want_state = scan_reference(v, True, ends)
    close(y.detach(), want_y, length)
    close(state.detach(), want_state, length)
    dx, ddelta = torch.autograd.grad((y, state), [g["x"], g["delta"]], [torch.ones_like(y), torch.ones_like(state)])
    assert torch.isfinite(dx).all() and torch.isfinite(ddelta).all()


@pytest.mark.parametrize("length", [0, 5, 300])
def test_scan_rates_of_infinity_do_not_touch_a_sequence_of_no_tokens(length):
    v = scan_inputs(64, 2, length, 24, 16)
    v["a"][3], v["a"][5, 2] = float("inf"), float("-inf")
    lengths = torch.zeros(2, dtype=torch.int32).cuda()
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, True, lengths, return_state=True)
    assert torch.equal(state.cpu(), v["state"]) and not y.any()
