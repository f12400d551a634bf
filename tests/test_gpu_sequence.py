"""The sequence operators on the GPU against their float64 definitions (oracle/sequence.py).

Tolerances.  One float32 operation is off by 2^-24 of its result, the special function unit's 2^x and
1/x by up to 2^-22.  A recurrence over T tokens adds at most T + 8 such steps of (2^-22 + 2 * 2^-24)
< 2^-21 each, so a float32 result is within (T + 8) 2^-21 of the largest value that takes part; a
gradient goes through four chained factors of that kind.  An output adds half a unit of its last
place: at most 2^-8 of the value in bfloat16 (8 bits of significand), 2^-11 in float16 (11 bits; 2^-25
near zero, in its subnormals).
"""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import ops
from oracle import sequence as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ROUNDING = {t: torch.finfo(t).eps / 2 for t in TYPES}  # of a value, at most: 2^-24, 2^-8, 2^-11


def close(actual, expected, steps, factor=1.0):
    """|actual - expected| <= factor steps 2^-21 max|expected| + half a last place of the value."""
    assert actual.shape == expected.shape
    actual64 = actual.double().cpu()
    if expected.numel() == 0:
        return
    assert torch.equal(torch.isfinite(actual64), torch.isfinite(expected))
    fine = torch.isfinite(expected)
    if not fine.any():
        return
    most = expected[fine].abs().max().item()
    room = factor * (steps + 8) * 2.0**-21 * most + ROUNDING[actual.dtype] * expected.abs() + 2.0**-25 * (actual.dtype == torch.float16)
    worst = ((actual64 - expected).abs() - room)[fine].max().item()
    assert worst <= 0, f"off by {worst} more than allowed (largest value {most})"


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (scale * torch.randn(*shape, generator=gen)).to(dtype)


def wide(t):
    return None if t is None else t.double()


def cuda(t):
    return None if t is None else t.cuda()


def scan_inputs(seed, batch, length, channels, states, groups=1, dtype=torch.float32, z=True, bias=True, d=True, state=True):
    gen = torch.Generator().manual_seed(seed)
    return {
        "x": randn(gen, batch, length, channels, dtype=dtype),
        "delta": randn(gen, batch, length, channels, dtype=dtype, scale=0.5),
        "a": -torch.arange(1, states + 1).float() * torch.exp(randn(gen, channels, states, scale=0.2)),
        "b": randn(gen, batch, length, groups, states, dtype=dtype),
        "c": randn(gen, batch, length, groups, states, dtype=dtype),
        "d": randn(gen, channels) if d else None,
        "z": randn(gen, batch, length, channels, dtype=dtype) if z else None,
        "delta_bias": randn(gen, channels, scale=0.5) - 2.0 if bias else None,
        "state": randn(gen, batch, channels, states) if state else None,
    }


def scan_reference(v, softplus, lengths=None):
    w = {k: wide(t) for k, t in v.items()}
    return oracle.selective_scan(
        w["x"], w["delta"], w["a"], w["b"], w["c"], w["d"], z=w["z"], delta_bias=w["delta_bias"], softplus=softplus,
        state=w["state"], lengths=lengths)


def scan_call(v, softplus, lengths=None, **more):
    return ops.selective_scan(
        v["x"], v["delta"], v["a"], v["b"], v["c"], v["d"], z=v["z"], delta_bias=v["delta_bias"], softplus=softplus,
        state=v["state"], lengths=lengths, **more)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "batch,length,channels,states,groups",
    [(1, 1, 1, 1, 1), (2, 33, 40, 16, 1), (1, 70, 24, 5, 2), (3, 31, 72, 33, 1), (1, 17, 200, 64, 1), (2, 64, 96, 20, 3),
     (1, 300, 9, 16, 1), (1, 1030, 33, 16, 1)],
)
def test_scan(dtype, batch, length, channels, states, groups):
    v = scan_inputs(length + channels, batch, length, channels, states, groups, dtype)
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, True, return_state=True)
    want_y, want_state = scan_reference(v, True)
    close(y, want_y, length)
    close(state, want_state, length)


@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("rest", [False, True])
def test_scan_optional_operands(z, rest):
    v = scan_inputs(3, 2, 45, 16, 8, 1, torch.float32, z=z, bias=rest, d=rest, state=rest)
    v["delta"] = v["delta"].abs() * 0.1
    if rest:  # no softplus: a negative sum would let the states grow without bound
        v["delta_bias"] = v["delta_bias"].abs() * 0.1
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, False, return_state=True)
    want_y, want_state = scan_reference(v, False)
    close(y, want_y, 45)
    close(state, want_state, 45)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [torch.int32, torch.int64])
def test_scan_ragged_ignores_what_lies_past_the_end(dtype, width):
    """Sequences of length 0, 1, around a tile's end and whole; NaN and infinity past the ends change nothing."""
    ends = [0, 1, 31, 32, 33, 100]
    v = scan_inputs(5, len(ends), 100, 24, 16, 1, dtype)
    want_y, want_state = scan_reference(v, True, ends)
    for name in ("x", "delta", "b", "c", "z"):
        for i, end in enumerate(ends):
            v[name][i, end:] = float("nan") if name in ("x", "b") else float("inf")
    y, state = scan_call(
        {k: cuda(t) for k, t in v.items()}, True, torch.tensor(ends, dtype=width).cuda(), return_state=True)
    close(y, want_y, 100)
    close(state, want_state, 100)
    assert torch.equal(state[0].cpu(), v["state"][0])
    for i, end in enumerate(ends):
        assert not y[i, end:].any()


def test_scan_of_no_tokens_keeps_the_state():
    v = scan_inputs(6, 2, 0, 8, 4)
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, True, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(state.cpu(), v["state"])
    v = scan_inputs(6, 0, 3, 8, 4)
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, True, return_state=True)
    assert y.shape == (0, 3, 8) and state.shape == (0, 8, 4)


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_scan_strided_operands(offset):
    """x and z as halves of one projection, b and c as parts of another, at aligned and odd places."""
    v = scan_inputs(7, 2, 40, 48, 16, 1, torch.bfloat16)
    want_y, _ = scan_reference(v, True)
    both = torch.zeros(2, 40, 2 * 48 + offset, dtype=torch.bfloat16).cuda()
    both[:, :, offset : offset + 48], both[:, :, offset + 48 :] = v["x"].cuda(), v["z"].cuda()
    rest = torch.zeros(2, 40, 32 + offset, dtype=torch.bfloat16).cuda()
    rest[:, :, offset : offset + 16], rest[:, :, offset + 16 :] = v["b"][:, :, 0].cuda(), v["c"][:, :, 0].cuda()
    w = {k: cuda(t) for k, t in v.items()}
    w["x"], w["z"] = both[:, :, offset : offset + 48], both[:, :, offset + 48 :]
    w["b"], w["c"] = rest[:, :, offset : offset + 16], rest[:, :, offset + 16 :]
    w["delta"] = w["delta"].transpose(0, 1).contiguous().transpose(0, 1)  # another order of the axes
    close(scan_call(w, True), want_y, 40)
    w["delta"] = w["delta"].transpose(1, 2).contiguous().transpose(1, 2)  # channels apart
    close(scan_call(w, True), want_y, 40)


def test_scan_in_two_calls_and_token_by_token():
    """A prompt at once, in two calls joined by the state, and as single tokens."""
    v = {k: cuda(t) for k, t in scan_inputs(8, 2, 50, 40, 16, 2).items()}
    whole, last = scan_call(v, True, return_state=True)
    cut = lambda s: {k: t[:, s] if t.dim() >= 3 and k != "state" else t for k, t in v.items()}  # noqa: E731
    first, state = scan_call(cut(slice(0, 19)), True, return_state=True)
    second, state2 = scan_call({**cut(slice(19, 50)), "state": state}, True, return_state=True)
    want, want_state = scan_reference({k: t.cpu() for k, t in v.items()}, True)
    close(torch.cat([first, second], 1), want, 50)
    close(state2, want_state, 50)
    state = v["state"].clone()
    rows = []
    for t in range(50):
        w = {k: u[:, t] for k, u in v.items() if u.dim() >= 3 and k != "state"}
        rows.append(ops.selective_scan_step(state, w["x"], w["delta"], v["a"], w["b"], w["c"], v["d"], z=w["z"],
                                            delta_bias=v["delta_bias"], softplus=True))
    close(torch.stack(rows, 1), want, 50)
    close(state, want_state, 50)
    close(whole, want, 50)
    close(last, want_state, 50)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("states", [1, 6, 16, 64, 128])
def test_scan_step(dtype, states):
    v = scan_inputs(9 + states, 5, 1, 27, states, 1, dtype)
    want_y, want_state = scan_reference(v, True)
    w = {k: cuda(t) for k, t in v.items()}
    y = ops.selective_scan_step(w["state"], w["x"][:, 0], w["delta"][:, 0], w["a"], w["b"][:, 0], w["c"][:, 0, 0], w["d"],
                                z=w["z"][:, 0], delta_bias=w["delta_bias"], softplus=True)
    close(y, want_y[:, 0], states)  # the sum over the states
    close(w["state"], want_state, 1)


def test_scan_extreme_delta():
    """softplus far out on both sides, decays that vanish and decays of one."""
    v = scan_inputs(10, 1, 12, 16, 4, 1, z=False, bias=False)
    v["delta"][0, :, :] = torch.tensor([-90.0, -20.0, -3.0, 0.0, 3.0, 19.9, 20.1, 60.0, 88.0, -1e-6, 1e-6, -45.0])[:, None]
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, True, return_state=True)
    want_y, want_state = scan_reference(v, True)
    close(y, want_y, 12)
    close(state, want_state, 12)


def grads_of(out, wanted, inputs):
    return torch.autograd.grad([o for o, w in zip(out, wanted) if w is not None], inputs, [w for w in wanted if w is not None])


def leaf(v, names):
    return {k: t.detach().clone().requires_grad_(k in names) if t is not None else None for k, t in v.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "batch,length,channels,states,groups,ends",
    [(1, 1, 3, 2, 1, None), (2, 37, 40, 16, 1, None), (1, 64, 24, 7, 2, None), (2, 50, 33, 30, 1, [50, 13]),
     (1, 20, 40, 64, 1, None), (3, 100, 17, 16, 1, [0, 1, 100]), (1, 400, 10, 16, 1, None)],
)
def test_scan_gradients(dtype, batch, length, channels, states, groups, ends):
    v = scan_inputs(20 + length, batch, length, channels, states, groups, dtype)
    names = list(v)
    gen = torch.Generator().manual_seed(1)
    dy, dstate = randn(gen, batch, length, channels, dtype=dtype), randn(gen, batch, channels, states)
    w = leaf({k: wide(t) for k, t in v.items()}, names)
    out = scan_reference(w, True, ends)
    want = dict(zip(names, grads_of(out, [wide(dy), wide(dstate)], [w[k] for k in names])))
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    lengths = None if ends is None else torch.tensor(ends, dtype=torch.int32).cuda()
    got = dict(zip(names, grads_of(scan_call(g, True, lengths, return_state=True), [cuda(dy), cuda(dstate)], [g[k] for k in names])))
    for k in names:
        # db and dc add up `channels`, the others up to batch * length terms
        close(got[k], want[k], length + (channels if k in "bc" else batch), factor=4.0)


@pytest.mark.parametrize("z", [False, True])
def test_scan_gradients_without_the_optional_operands(z):
    v = scan_inputs(31, 2, 40, 16, 16, 1, torch.float32, z=z, bias=False, d=False, state=False)
    v["delta"] = v["delta"].abs() * 0.1
    names = [k for k, t in v.items() if t is not None]
    dy = randn(torch.Generator().manual_seed(2), 2, 40, 16)
    w = leaf({k: wide(t) for k, t in v.items()}, names)
    want = torch.autograd.grad(scan_reference(w, False)[0], [w[k] for k in names], wide(dy))
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    got = torch.autograd.grad(scan_call(g, False), [g[k] for k in names], cuda(dy))
    for a, b in zip(got, want):
        close(a, b, 40, factor=4.0)


def test_scan_gradients_of_expanded_inputs():
    """b and c shared by the batch (expanded): their gradients add up over it."""
    v = scan_inputs(32, 3, 21, 16, 16)
    names = ["b", "c"]
    dy = randn(torch.Generator().manual_seed(3), 3, 21, 16)
    w = leaf({k: wide(t[:1]) if k in names else wide(t) for k, t in v.items()}, names)
    g = leaf({k: cuda(t[:1]) if k in names else cuda(t) for k, t in v.items()}, names)
    spread = lambda q: {k: t.expand(3, -1, -1, -1) if k in names else t for k, t in q.items()}  # noqa: E731
    want = torch.autograd.grad(scan_reference(spread(w), True)[0], [w[k] for k in names], wide(dy))
    got = torch.autograd.grad(scan_call(spread(g), True), [g[k] for k in names], cuda(dy))
    for a, b in zip(got, want):
        close(a, b, 21 + 3 * 16, factor=4.0)


def against_differences(loss, values, grads, seed):
    """<grad, v> against the central difference of the float64 loss along random directions v.  Rounding
    of the loss: 2^-50 |loss| / eps; truncation: eps^2 times a third derivative; eps = 1e-4."""
    gen = torch.Generator().manual_seed(seed)
    for name, grad in grads.items():
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        v /= v.norm()
        eps = 1e-4
        ends = [loss({**values, name: values[name] + sign * eps * v}).item() for sign in (1.0, -1.0)]
        slope = (ends[0] - ends[1]) / (2 * eps)
        along = (grad.double().cpu() * v).sum().item()
        assert abs(along - slope) <= 1e-4 * grad.double().norm().item() + 1e-6 * (1 + abs(ends[0])), name


def test_scan_gradients_against_differences():
    v = scan_inputs(33, 2, 30, 12, 8, 2)
    names = list(v)
    gen = torch.Generator().manual_seed(4)
    dy, dstate = randn(gen, 2, 30, 12), randn(gen, 2, 12, 8)
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    got = grads_of(scan_call(g, True, return_state=True), [cuda(dy), cuda(dstate)], [g[k] for k in names])

    def loss(w):
        y, state = scan_reference(w, True)
        return (y * dy).sum() + (state * dstate).sum()

    against_differences(loss, {k: wide(t) for k, t in v.items()}, dict(zip(names, got)), 5)


def test_scan_results_do_not_vary():
    """The same call gives the same bits, on another stream too."""
    v = scan_inputs(34, 2, 300, 64, 16, 1, torch.bfloat16)
    names = list(v)
    dy = randn(torch.Generator().manual_seed(6), 2, 300, 64, dtype=torch.bfloat16).cuda()
    runs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            g = leaf({k: cuda(t) for k, t in v.items()}, names)
            y = scan_call(g, True)
            runs.append([y.detach(), *torch.autograd.grad(y, [g[k] for k in names], dy)])
        stream.synchronize()
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# ---------------------------------------------------------------------------
# convolution


def conv_inputs(seed, batch, length, channels, width, dtype, bias=True, state=True):
    gen = torch.Generator().manual_seed(seed)
    return {
        "x": randn(gen, batch, length, channels, dtype=dtype),
        "weight": randn(gen, channels, width),
        "bias": randn(gen, channels) if bias else None,
        "state": randn(gen, batch, width - 1, channels, dtype=dtype) if state else None,
    }


def conv_reference(v, activation, lengths=None):
    return oracle.causal_conv1d(v["x"], v["weight"], v["bias"], activation=activation, state=v["state"], lengths=lengths)


def conv_call(v, activation, lengths=None, return_state=True):
    return ops.causal_conv1d(v["x"], v["weight"], v["bias"], activation=activation, state=v["state"], lengths=lengths,
                             return_state=return_state)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4])
@pytest.mark.parametrize("batch,length,channels", [(1, 1, 1), (2, 2, 24), (3, 130, 40), (1, 37, 13), (1, 9, 1030)])
def test_conv(dtype, width, batch, length, channels):
    v = conv_inputs(length + width, batch, length, channels, width, dtype)
    y, state = conv_call({k: cuda(t) for k, t in v.items()}, "silu")
    want_y, want_state = conv_reference({k: wide(t) for k, t in v.items()}, "silu")
    close(y, want_y, width)
    assert torch.equal(state.double().cpu(), want_state)


def test_conv_optional_operands_and_strides():
    v = conv_inputs(1, 2, 20, 24, 4, torch.bfloat16, bias=False, state=False)
    want, _ = conv_reference({k: wide(t) for k, t in v.items()}, None)
    for offset in (0, 3, 8):
        part = torch.zeros(2, 20, 50, dtype=torch.bfloat16).cuda()
        part[:, :, offset : offset + 24] = v["x"].cuda()
        y = ops.causal_conv1d(part[:, :, offset : offset + 24], v["weight"].cuda())
        close(y, want, 4)
    y = ops.causal_conv1d(v["x"].cuda().transpose(1, 2).contiguous().transpose(1, 2), v["weight"].cuda())
    close(y, want, 4)


@pytest.mark.parametrize("width", [2, 4])
def test_conv_ragged_ignores_what_lies_past_the_end(width):
    ends = [0, 1, 2, 5, 64, 129, 200]
    v = conv_inputs(2, len(ends), 200, 16, width, torch.float32)
    want_y, want_state = conv_reference({k: wide(t) for k, t in v.items()}, "silu", ends)
    for i, end in enumerate(ends):
        v["x"][i, end:] = float("nan")
    y, state = conv_call({k: cuda(t) for k, t in v.items()}, "silu", torch.tensor(ends).cuda())
    close(y, want_y, width)
    assert torch.equal(state.double().cpu(), want_state)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4])
def test_conv_step(dtype, width):
    """Token by token against the whole sequence, the state shifted in place."""
    v = conv_inputs(3 + width, 3, 9, 21, width, dtype)
    want_y, want_state = conv_reference({k: wide(t) for k, t in v.items()}, "silu")
    w = {k: cuda(t) for k, t in v.items()}
    rows = [ops.causal_conv1d_step(w["state"], w["x"][:, t], w["weight"], w["bias"], activation="silu") for t in range(9)]
    close(torch.stack(rows, 1), want_y, width)
    assert torch.equal(w["state"].double().cpu(), want_state)


def test_conv_of_no_tokens():
    v = conv_inputs(4, 2, 0, 8, 4, torch.float32)
    y, state = conv_call({k: cuda(t) for k, t in v.items()}, "silu")
    assert y.shape == (2, 0, 8) and torch.equal(state.cpu(), v["state"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4])
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("batch,length,channels,ends", [(1, 1, 5, None), (2, 150, 24, None), (3, 70, 13, [0, 2, 70])])
def test_conv_gradients(dtype, width, activation, batch, length, channels, ends):
    v = conv_inputs(40 + length, batch, length, channels, width, dtype)
    names = list(v)
    gen = torch.Generator().manual_seed(7)
    dy, dstate = randn(gen, batch, length, channels, dtype=dtype), randn(gen, batch, width - 1, channels, dtype=dtype)
    w = leaf({k: wide(t) for k, t in v.items()}, names)
    wanted = [wide(dy), wide(dstate) if width > 1 else None]
    out = conv_reference(w, activation, ends)
    want = torch.autograd.grad([o for o, q in zip(out, wanted) if q is not None], [w[k] for k in names],
                               [q for q in wanted if q is not None], allow_unused=True)
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    lengths = None if ends is None else torch.tensor(ends).cuda()
    got = grads_of(conv_call(g, activation, lengths), [cuda(dy), cuda(dstate) if width > 1 else None], [g[k] for k in names])
    for k, a, b in zip(names, got, want):
        # the parameters' gradients add up batch * length terms
        close(a, torch.zeros_like(w[k]) if b is None else b, width + (batch * length if k in ("weight", "bias") else 0), factor=4.0)


def test_conv_gradients_against_differences():
    v = conv_inputs(50, 2, 12, 10, 3, torch.float32)
    names = list(v)
    gen = torch.Generator().manual_seed(8)
    dy, dstate = randn(gen, 2, 12, 10), randn(gen, 2, 2, 10)
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    got = grads_of(conv_call(g, "silu"), [cuda(dy), cuda(dstate)], [g[k] for k in names])

    def loss(w):
        y, state = conv_reference(w, "silu")
        return (y * dy).sum() + (state * dstate).sum()

    against_differences(loss, {k: wide(t) for k, t in v.items()}, dict(zip(names, got)), 9)


# ---------------------------------------------------------------------------
# norm


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 7), (5, 64), (33, 250), (2, 2048), (3, 5003), (2, 12288), (1, 40000)])
@pytest.mark.parametrize("residual", [None, "same", "wide"])
def test_norm(dtype, rows, columns, residual):
    gen = torch.Generator().manual_seed(columns)
    x, weight = randn(gen, rows, columns, dtype=dtype), randn(gen, columns)
    r = None if residual is None else randn(gen, rows, columns, dtype=dtype if residual == "same" else torch.float32)
    want_y, want_s = oracle.rms_norm(x.double(), weight.double(), wide(r))
    got = ops.rms_norm(x.cuda(), weight.cuda(), residual=cuda(r))
    # sums of `columns` squares in a tree: a few dozen roundings
    if r is None:
        close(got, want_y, 24)
    else:
        close(got[0], want_y, 24)
        close(got[1], want_s, 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns", [65, 127, 1001, 2052, 9003])
def test_norm_of_rows_that_drift_past_the_boundaries(dtype, columns):
    """Odd numbers of columns: every row starts elsewhere within a vector, its ends beside its neighbours'."""
    gen = torch.Generator().manual_seed(columns)
    x, r, weight = randn(gen, 19, columns, dtype=dtype), randn(gen, 19, columns, dtype=dtype), randn(gen, columns)
    want_y, want_s = oracle.rms_norm(x.double(), weight.double(), r.double())
    y, s = ops.rms_norm(x.cuda(), weight.cuda(), residual=r.cuda())
    close(y, want_y, 24)
    close(s, want_s, 0)
    wide_y, wide_s = ops.rms_norm(x.cuda(), weight.cuda().to(dtype), residual=r.cuda().float())
    close(wide_y, oracle.rms_norm(x.double(), weight.to(dtype).double(), r.double())[0], 24)
    close(wide_s, want_s, 0)
    q, scale, _ = ops.rms_norm(x.cuda(), weight.cuda(), residual=r.cuda(), quantize="int8")
    want_scale = want_y.abs().amax(1) / 127.0
    assert ((q.double().cpu() - want_y / want_scale[:, None]).abs() <= 0.5 + 64 * 2.0**-21 * 127.0).all()
    assert ((scale.double().cpu() - want_scale).abs() <= 32 * 2.0**-21 * want_scale).all()


@pytest.mark.parametrize("quantize,most,step", [("e4m3", 448.0, 2.0**-4), ("int8", 127.0, None)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 16), (4, 100), (70, 96), (2, 4096), (3, 9000)])
def test_norm_in_8_bits(quantize, most, step, dtype, rows, columns):
    gen = torch.Generator().manual_seed(rows + columns)
    x, r, weight = randn(gen, rows, columns, dtype=dtype), randn(gen, rows, columns, dtype=dtype), randn(gen, columns)
    want_y, want_s = oracle.rms_norm(x.double(), weight.double(), r.double())
    q, scale, s = ops.rms_norm(x.cuda(), weight.cuda(), residual=r.cuda(), quantize=quantize)
    close(s, want_s, 0)
    want_scale = want_y.abs().amax(1) / most
    assert ((scale.double().cpu() - want_scale).abs() <= 32 * 2.0**-21 * want_scale).all()
    # half a step of the format at the value's size (e4m3: 2^-4 of it, at least 2^-10; int8: 1/2), and the
    # float32 errors of the value and the scale
    exact = want_y / want_scale[:, None]
    half = torch.clamp(exact.abs() * step, min=2.0**-10) if step else torch.full_like(exact, 0.5)
    assert ((q.double().cpu() - exact).abs() <= half + 64 * 2.0**-21 * most).all()
    assert q.double().abs().amax(1).eq(most).all()


def test_norm_of_special_rows():
    """A zero row, a tiny one, a NaN and an infinity: each row for itself."""
    x = torch.ones(5, 40)
    x[0], x[1], x[2, 3], x[3, 5] = 0.0, 1e-30, float("nan"), float("inf")
    y = ops.rms_norm(x.cuda()).cpu()
    assert not y[0].any() and torch.isnan(y[2]).all() and torch.isnan(y[3, 5])
    close(y[4:], oracle.rms_norm(x[4:].double())[0], 24)
    close(y[1:2], oracle.rms_norm(x[1:2].double())[0], 24)
    for quantize in ("e4m3", "int8"):
        q, scale = ops.rms_norm(x.cuda(), quantize=quantize)
        assert not q[0].float().any() and scale[0].item() == 2.0**-126
        assert torch.isnan(scale[2]) and torch.isnan(scale[3])
        assert torch.isfinite(scale[4]) and q[4].float().abs().eq(448.0 if quantize == "e4m3" else 127.0).all()


def test_norm_strided_rows_and_ranks():
    gen = torch.Generator().manual_seed(11)
    x = randn(gen, 3, 5, 96)
    want = oracle.rms_norm(x.double())[0]
    part = torch.zeros(3, 5, 130).cuda()
    part[:, :, 3:99] = x.cuda()
    close(ops.rms_norm(part[:, :, 3:99]), want, 24)
    close(ops.rms_norm(x.cuda().transpose(1, 2).contiguous().transpose(1, 2)), want, 24)
    close(ops.rms_norm(x.cuda()[0, 0]), want[0, 0], 24)
    assert ops.rms_norm(torch.zeros(0, 8).cuda()).shape == (0, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 5), (700, 40), (19, 1030), (5, 6000), (3, 20000)])
@pytest.mark.parametrize("residual", [None, "same", "wide"])
def test_norm_gradients(dtype, rows, columns, residual):
    gen = torch.Generator().manual_seed(columns + 1)
    x, weight, dy = randn(gen, rows, columns, dtype=dtype), randn(gen, columns), randn(gen, rows, columns, dtype=dtype)
    r = ds = None
    if residual is not None:
        kind = dtype if residual == "same" else torch.float32
        r, ds = randn(gen, rows, columns, dtype=kind), randn(gen, rows, columns, dtype=kind)
    inputs = [x, weight] + ([r] if r is not None else [])
    w = [t.double().requires_grad_() for t in inputs]
    out = oracle.rms_norm(w[0], w[1], w[2] if r is not None else None)
    want = grads_of(out, [dy.double(), wide(ds)], w)
    g = [t.cuda().requires_grad_() for t in inputs]
    got = ops.rms_norm(g[0], g[1], residual=g[2] if r is not None else None)
    got = grads_of(got if r is not None else (got,), [dy.cuda(), cuda(ds)], g)
    for k, (a, b) in enumerate(zip(got, want)):
        close(a, b, 24 + (rows if k == 1 else 0), factor=4.0)


def test_norm_gradients_against_differences():
    gen = torch.Generator().manual_seed(12)
    v = {"x": randn(gen, 6, 50), "weight": randn(gen, 50), "residual": randn(gen, 6, 50)}
    dy, ds = randn(gen, 6, 50), randn(gen, 6, 50)
    g = leaf({k: cuda(t) for k, t in v.items()}, list(v))
    got = grads_of(ops.rms_norm(g["x"], g["weight"], residual=g["residual"]), [dy.cuda(), ds.cuda()], list(g.values()))

    def loss(w):
        y, s = oracle.rms_norm(w["x"], w["weight"], w["residual"])
        return (y * dy).sum() + (s * ds).sum()

    against_differences(loss, {k: wide(t) for k, t in v.items()}, dict(zip(v, got)), 13)


# ---------------------------------------------------------------------------
# 4-bit weights


def int4_inputs(seed, inputs, outputs, group, zeros, scale_dtype):
    gen = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (outputs, inputs // 2), generator=gen, dtype=torch.uint8)
    scales = (0.5 + torch.rand(outputs, inputs // group, generator=gen)).to(scale_dtype)
    z = torch.randint(0, 16, (outputs, inputs // group), generator=gen, dtype=torch.uint8) if zeros else None
    return gen, packed, scales, z


def int4_close(y, x, packed, scales, zeros, x_scale=None):
    """Products are exact; sums of K float32 terms and the groups' scales are off by at most (K / 16 + 8) 2^-23 of the
    sum of the terms' sizes (the tensor core adds sixteen products at a time, and may cut instead of rounding)."""
    w = oracle.int4_weight(packed, scales, zeros)
    xs = x.double() if x.dtype != torch.float8_e4m3fn else x.float().double()
    if x_scale is not None:
        xs = xs * x_scale.double()[..., None]
    want, size = xs @ w.t(), xs.abs() @ w.t().abs()
    room = (w.shape[1] / 16 + 8) * 2.0**-23 * size + ROUNDING[y.dtype] * want.abs()
    assert y.shape == want.shape
    worst = ((y.double().cpu() - want).abs() - room).max().item()
    assert worst <= 0, worst


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    "rows,inputs,outputs,group,zeros",
    [(1, 32, 1, 32, False), (1, 256, 100, 128, True), (5, 1056, 67, 32, True), (8, 512, 16, 64, False), (9, 640, 130, 128, True),
     (17, 192, 33, 96, True), (33, 1024, 40, 256, False), (64, 128, 17, 128, True), (70, 320, 50, 64, True), (1, 8192, 48, 128, False),
     (3, 18432, 20, 64, True)],
)
def test_int4(dtype, rows, inputs, outputs, group, zeros):
    gen, packed, scales, z = int4_inputs(rows + inputs, inputs, outputs, group, zeros, torch.float32 if dtype == torch.float32 else dtype)
    x = randn(gen, rows, inputs, dtype=dtype)
    y = ops.int4_linear(x.cuda(), packed.cuda(), scales.cuda(), cuda(z))
    assert y.dtype == dtype
    int4_close(y, x, packed, scales, z)


@pytest.mark.parametrize("quantize", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,inputs,outputs,group", [(1, 256, 30, 128), (12, 1024, 70, 64), (40, 352, 33, 32)])
@pytest.mark.parametrize("dtype", [None, torch.float32, torch.float16])
def test_int4_of_the_norm_in_8_bits(quantize, rows, inputs, outputs, group, dtype):
    gen, packed, scales, z = int4_inputs(rows, inputs, outputs, group, True, torch.bfloat16)
    q, scale = ops.rms_norm(randn(gen, rows, inputs, dtype=torch.bfloat16).cuda(), quantize=quantize)
    y = ops.int4_linear(q, packed.cuda(), scales.cuda(), z.cuda(), x_scale=scale, dtype=dtype)
    assert y.dtype == (dtype or torch.bfloat16)
    int4_close(y, q.cpu(), packed, scales, z, scale.cpu())


def test_int4_float32_activations_are_exact_parts():
    """Values whose significands use all 24 bits, huge ones and tiny ones, one at a time: the product is the float32 value."""
    values = torch.tensor([1.0 + 2.0**-23, 3.3333333, 16777215.0, 3.0e38, 1.7e-30, -2.0**-100 * 1.2345678, 0.0])
    x = torch.zeros(len(values), 64)
    x[torch.arange(len(values)), torch.arange(len(values)) * 9] = values
    packed = ops.int4_pack(torch.full((3, 64), 9, dtype=torch.uint8))  # weight 1
    y = ops.int4_linear(x.cuda(), packed.cuda(), torch.ones(3, 2).cuda()).cpu()
    assert torch.equal(y, values[:, None].expand(-1, 3))


def test_int4_nonfinite_activations_stay_in_their_row():
    gen, packed, scales, _ = int4_inputs(1, 128, 20, 64, False, torch.float32)
    for dtype in TYPES:
        x = randn(gen, 4, 128, dtype=dtype)
        clean = ops.int4_linear(x.cuda(), packed.cuda(), scales.to(dtype).cuda()).cpu()
        x[1, 7], x[2, 9] = float("nan"), float("inf")
        y = ops.int4_linear(x.cuda(), packed.cuda(), scales.to(dtype).cuda()).cpu()
        assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
        assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()


def test_int4_shapes_and_strides():
    gen, packed, scales, z = int4_inputs(2, 256, 24, 64, True, torch.bfloat16)
    x = randn(gen, 2, 3, 300, dtype=torch.bfloat16)
    part = x.cuda()[:, :, 5:261]
    y = ops.int4_linear(part, packed.cuda(), scales.cuda(), z.cuda())
    int4_close(y, x[:, :, 5:261], packed, scales, z)
    room = torch.zeros(24, 129, dtype=torch.uint8).cuda()
    room[:, 1:] = packed.cuda()
    int4_close(ops.int4_linear(part, room[:, 1:], scales.cuda(), z.cuda()), x[:, :, 5:261], packed, scales, z)
    assert ops.int4_linear(part[:, :0], packed.cuda(), scales.cuda()).shape == (2, 0, 24)
    assert ops.int4_linear(part[0, 0], packed.cuda(), scales.cuda()).shape == (24,)


@pytest.mark.parametrize("symmetric", [True, False])
def test_int4_quantize(symmetric):
    """Each weight is within half a step of its code's value, and the product follows."""
    gen = torch.Generator().manual_seed(3)
    w = randn(gen, 40, 256)
    packed, scales, zeros = ops.int4_quantize(w.cuda(), 64, symmetric=symmetric)
    back = oracle.int4_weight(packed.cpu(), scales.cpu(), None if zeros is None else zeros.cpu())
    step = scales.double().cpu().repeat_interleave(64, 1)
    # a whole zero point moves an asymmetric group's ends by up to half a step more
    assert ((back - w.double()).abs() <= (0.5 if symmetric else 1.0) * step * (1 + 2.0**-20)).all()
    x = randn(gen, 2, 256)
    int4_close(ops.int4_linear(x.cuda(), packed, scales, zeros), x, packed.cpu(), scales.cpu(), None if zeros is None else zeros.cpu())


def test_strides_past_32_bits():
    """Two rows 2^31 elements apart: the second one's offset does not fit 32 bits."""
    far = 2**31
    base = torch.empty(far + 4096, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator().manual_seed(13)

    def spread(t):
        view = base.as_strided(t.shape, (far, *t.stride()[1:]))
        view.copy_(t.cuda())
        return view

    v = scan_inputs(14, 2, 9, 24, 16, 1, torch.bfloat16)
    want, want_state = scan_reference(v, True)
    w = {k: cuda(t) for k, t in v.items()}
    for name in ("x", "delta", "z", "b", "c"):
        y, state = scan_call({**w, name: spread(v[name])}, True, return_state=True)
        close(y, want, 9)
        close(state, want_state, 9)
    x, weight = randn(gen, 2, 9, 24, dtype=torch.bfloat16), randn(gen, 24, 4)
    close(ops.causal_conv1d(spread(x), weight.cuda()), oracle.causal_conv1d(x.double(), weight.double())[0], 4)
    rows = randn(gen, 2, 256, dtype=torch.bfloat16)
    close(ops.rms_norm(spread(rows)), oracle.rms_norm(rows.double())[0], 24)
    _, packed, scales, z = int4_inputs(15, 256, 20, 64, True, torch.bfloat16)
    int4_close(ops.int4_linear(spread(rows), packed.cuda(), scales.cuda(), z.cuda()), rows, packed, scales, z)


@pytest.mark.parametrize("length,channels", [(700, 7), (2100, 20)])
def test_scan_gradients_of_a_split_length(length, channels):
    """Few channels: the length is run in segments, whose states and adjoints are joined."""
    v = scan_inputs(16, 1, length, channels, 5)
    names = list(v)
    gen = torch.Generator().manual_seed(17)
    dy, dstate = randn(gen, 1, length, channels), randn(gen, 1, channels, 5)
    ends = torch.tensor([length - 150])
    w = leaf({k: wide(t) for k, t in v.items()}, names)
    want = grads_of(scan_reference(w, True, ends), [wide(dy), wide(dstate)], [w[k] for k in names])
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    got = grads_of(scan_call(g, True, ends.cuda(), return_state=True), [cuda(dy), cuda(dstate)], [g[k] for k in names])
    for k, a, b in zip(names, got, want):
        close(a, b, length + channels, factor=4.0)
