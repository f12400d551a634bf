"""Errors of the sequence operators that would add up: means over many results, long sums, and single functions.

Random errors of a float32 result are below 2^-24 of it; what the tests here look for is larger or has a mean.
"""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import ops

pytestmark = pytest.mark.gpu


def decays(seed, batch, length, channels):
    """Step sizes that make a state's exponents (base 2) lie between -0.01 and -0.001, and its logarithm after them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    delta = (0.001 + 0.009 * torch.rand(batch, length, channels, generator=gen, device="cuda")) * 0.6931
    return delta, -delta.double().sum(1)


def mean_error(actual, log_expected):
    return (actual.double() * torch.exp(-log_expected) - 1.0).mean().item()


@pytest.mark.parametrize("batch,channels", [(3, 4096), (2, 96)])
def test_scan_decays_have_no_bias(batch, channels):
    """A state that only decays, forwards and (its gradient) backwards: exponentials rounded to nearest would have errors up
    to 2^-25 of either sign; their mean over all channels stays below a quarter of that per token, 2^-27.  Whole
    sequences (many channels) and ones run in segments (few)."""
    length = 2048
    delta, log_state = decays(1, batch, length, channels)
    zero, none = torch.zeros_like(delta), torch.zeros(batch, length, 1, device="cuda")
    a = -torch.ones(channels, 1, device="cuda")
    state = torch.ones(batch, channels, 1, device="cuda", requires_grad=True)
    _, last = ops.selective_scan(zero, delta, a, none, none, state=state, return_state=True)
    assert abs(mean_error(last.detach()[..., 0], log_state)) <= length * 2.0**-27
    (grad,) = torch.autograd.grad(last, state, torch.ones_like(last))
    assert abs(mean_error(grad[..., 0], log_state)) <= length * 2.0**-27


def test_step_decays_have_no_bias():
    length, channels = 256, 4096
    delta, log_state = decays(2, 8, length, channels)
    zero, none = torch.zeros(8, channels, device="cuda"), torch.zeros(8, 1, device="cuda")
    a = -torch.ones(channels, 1, device="cuda")
    state = torch.ones(8, channels, 1, device="cuda")
    for t in range(length):
        ops.selective_scan_step(state, zero, delta[:, t], a, none, none)
    assert abs(mean_error(state[..., 0], log_state)) <= length * 2.0**-27


@pytest.mark.parametrize("rate", [-1.0, -1e30, 3.0])
def test_a_step_size_of_zero_keeps_the_state_exactly(rate):
    gen = torch.Generator(device="cuda").manual_seed(3)
    state = torch.randn(2, 40, 16, generator=gen, device="cuda")
    zero, bc = torch.zeros(2, 50, 40, device="cuda"), torch.ones(2, 50, 16, device="cuda")
    a = torch.full((40, 16), rate, device="cuda")
    _, last = ops.selective_scan(zero, zero, a, bc, bc, state=state, return_state=True)
    assert torch.equal(last, state)
    held = state.clone()
    ops.selective_scan_step(held, zero[:, 0], zero[:, 0], a, bc[:, 0], bc[:, 0])
    assert torch.equal(held, state)


def relative(actual, expected):
    return ((actual.double() - expected).norm() / expected.norm()).item()


def test_scan_sums_over_a_long_length():
    """dD and d(delta_bias) over 16384 tokens that are not split.  A running float32 sum of n terms of either sign is off by at
    most about 2^-25 sqrt(n / 2) of itself; sums of sums of 64 terms, 32 of them, over 8 threads and 32 sequences by
    2^-25 sqrt(32 + 16 + 4 + 16), in round figures 12 2^-25.  One running sum: 32 2^-25 and more."""
    batch, length, channels = 32, 16384, 320
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.randn(batch, length, channels, generator=gen, device="cuda") for _ in range(2))
    delta = (0.1 * torch.rand(batch, length, channels, generator=gen, device="cuda")).requires_grad_()
    bc = torch.randn(2, batch, length, 1, generator=gen, device="cuda")
    a = -torch.ones(channels, 1, device="cuda")
    d, bias = torch.ones(channels, device="cuda", requires_grad=True), torch.zeros(channels, device="cuda", requires_grad=True)
    y = ops.selective_scan(x, delta, a, bc[0], bc[1], d, delta_bias=bias)
    ddelta, dd, dbias = torch.autograd.grad(y, [delta, d, bias], dy)
    assert relative(dd, sum((x[i].double() * dy[i].double()).sum(0) for i in range(batch))) <= 12 * 2.0**-25
    assert relative(dbias, sum(ddelta[i].double().sum(0) for i in range(batch))) <= 12 * 2.0**-25


@pytest.mark.parametrize("rows,columns", [(1 << 24, 32), (3 << 20, 33)])
def test_norm_sums_over_many_rows(rows, columns):
    """dweight over millions of rows, in float32 sums of at most 64 rows, sums of these, and the blocks' sums: by the measure
    above 2^-25 sqrt(32 + 32 + 64).  One running sum of a slot's 2000 to 3500 rows: 2^-25 sqrt(1000) and more."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, dy = (torch.randn(rows, columns, generator=gen, device="cuda") for _ in range(2))
    weight = torch.ones(columns, device="cuda", requires_grad=True)
    (dweight,) = torch.autograd.grad(ops.rms_norm(x, weight), weight, dy)
    want = 0.0
    for part, grad in zip(x.chunk(16), dy.chunk(16)):
        part = part.double()
        want = want + (grad.double() * part * torch.rsqrt((part * part).mean(1, keepdim=True) + 1e-6)).sum(0)
    assert relative(dweight, want) <= 12 * 2.0**-25


def test_norm_sums_of_columns_over_rows_by_element_and_in_vectors():
    """More than 64 rows to a slot in every width of the kernels, each column's sum by itself: all dy of one sign."""
    for columns in (8, 33, 1000, 3000, 9001):
        rows = 148 * 70 * max(1, 8 * 256 // columns)
        gen = torch.Generator(device="cuda").manual_seed(columns)
        x = torch.rand(rows, columns, generator=gen, device="cuda") + 0.5
        weight = torch.ones(columns, device="cuda", requires_grad=True)
        (dweight,) = torch.autograd.grad(ops.rms_norm(x, weight), weight, torch.ones_like(x))
        want = 0.0
        for part in x.chunk(8):
            part = part.double()
            want = want + (part * torch.rsqrt((part * part).mean(1, keepdim=True) + 1e-6)).sum(0)
        # terms of one sign: up to 2^-25 per addition on average, of 64 + rows / slots / 64 + blocks' rows / 32 + 5
        assert ((dweight.double() - want).abs() <= 256 * 2.0**-24 * want).all(), columns


def test_softplus_keeps_small_results():
    """A step's softplus seen through a state of no decay: 2^x is off by up to 2^-22 of itself, the rounding of v log2(e) in
    front of it by 2^-23.7 |v|, the polynomial by 7.6e-8 and its evaluation by 2^-23: in all within 2^-21 + |v| 2^-23."""
    v = torch.cat([torch.linspace(-80, 30, 40000), torch.tensor([-1e-6, 0.0, 1e-6, 19.9, 20.1, 80.0])]).cuda()
    one, none = torch.ones(1, v.numel(), device="cuda"), torch.zeros(1, 1, device="cuda")
    want = torch.nn.functional.softplus(v.double(), threshold=60.0)
    room = (2.0**-21 + v.double().abs() * 2.0**-23) * want
    zero = torch.zeros(v.numel(), 1, device="cuda")
    _, state = ops.selective_scan(one[:, None], v[None, None], zero, none[:, None] + 1, none[:, None], softplus=True, return_state=True)
    assert ((state[0, :, 0].double() - want).abs() <= room).all()
    held = torch.zeros(1, v.numel(), 1, device="cuda")
    ops.selective_scan_step(held, one, v[None], zero, none + 1, none, softplus=True)
    assert ((held[0, :, 0].double() - want).abs() <= room).all()
