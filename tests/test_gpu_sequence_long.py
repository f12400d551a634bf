"""The sequence operators at sizes where their kernels run for many turns, against their float64 definitions.

Tolerances as in test_gpu_sequence.py, whose helpers and derivations these are.
"""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import _lib, ops, sequence
from test_gpu_sequence import (
    TYPES,
    close,
    cuda,
    grads_of,
    int4_close,
    int4_inputs,
    leaf,
    randn,
    scan_call,
    scan_inputs,
    scan_reference,
    wide,
)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,inputs,outputs", [(torch.float32, 1280, 7), (torch.bfloat16, 64, 5), (torch.float8_e4m3fn, 96, 3)])
def test_int4_of_more_rows_than_a_grid_holds(dtype, inputs, outputs):
    """70001 rows, the first of them with k in parts."""
    gen, packed, scales, z = int4_inputs(21, inputs, outputs, 32, True, torch.float32)
    x = randn(gen, 70001, inputs, dtype=dtype)
    x_scale = 0.5 + torch.rand(70001, generator=gen) if dtype == torch.float8_e4m3fn else None
    y = ops.int4_linear(x.cuda(), packed.cuda(), scales.cuda(), z.cuda(), x_scale=cuda(x_scale), dtype=torch.float32)
    int4_close(y, x, packed, scales, z, x_scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_int4_in_slices(dtype):
    """A prompt whose partial sums would need gigabytes at once: every slice's rows, at the seams too."""
    rows, inputs, outputs = 12000, 9000 // 32 * 32, 2051
    gen, packed, scales, _ = int4_inputs(22, inputs, outputs, 32, False, dtype)
    x = randn(gen, rows, inputs, dtype=dtype)
    y = ops.int4_linear(x.cuda(), packed.cuda(), scales.cuda())
    size = _lib.load().xe_int4_linear_workspace_size(rows, inputs, outputs, _lib.XE_F32 if dtype == torch.float32 else _lib.XE_BF16)
    assert 0 < size <= 512 << 20
    some = torch.cat([torch.arange(0, rows, 61), torch.arange(rows - 70, rows)])
    int4_close(y[some.cuda()], x[some], packed, scales, None)


# ---------------------------------------------------------------------------
# norm: more rows than the device holds at once, so that a block's rings, reduction buffers and sums go round


def excess(actual, expected, dtype, steps, terms=0.0):
    """As test_gpu_sequence.close, on the GPU (float64 there): the largest excess over the allowed error."""
    rounding = torch.finfo(dtype).eps / 2
    room = (steps + 8) * 2.0**-21 * expected.abs().max() + rounding * expected.abs() + 2.0**-25 * (dtype == torch.float16) + terms
    return ((actual.double() - expected).abs() - room).max().item()


NORM_SHAPES = [(6001, 96), (1500, 2560), (1500, 2563), (700, 4096), (450, 9000), (450, 12288), (400, 20000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", NORM_SHAPES)
@pytest.mark.parametrize("wide", [False, True])
def test_norm_of_many_rows(dtype, rows, columns, wide):
    gen = torch.Generator(device="cuda").manual_seed(columns)
    x, r = (torch.randn(rows, columns, generator=gen, device="cuda", dtype=torch.float32).to(dtype) for _ in range(2))
    if wide:
        r = r.float()
    weight = torch.randn(columns, generator=gen, device="cuda")
    s = x.double() + r.double()
    want = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * weight.double()
    y, total = ops.rms_norm(x, weight, residual=r)
    assert excess(y, want, dtype, 24) <= 0
    assert excess(total, s, r.dtype, 0) <= 0
    plain = x.double() * torch.rsqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6)
    assert excess(ops.rms_norm(x), plain, dtype, 24) <= 0
    for quantize, most in (("e4m3", 448.0), ("int8", 127.0)):
        q, scale, again = ops.rms_norm(x, weight, residual=r, quantize=quantize)
        want_scale = want.abs().amax(1) / most
        assert torch.equal(again, total)
        assert ((scale.double() - want_scale).abs() <= 32 * 2.0**-21 * want_scale).all()
        exact = want / want_scale[:, None]
        half = torch.clamp(exact.abs() * 2.0**-4, min=2.0**-10) if quantize == "e4m3" else torch.full_like(exact, 0.5)
        assert ((q.double() - exact).abs() <= half + 64 * 2.0**-21 * most).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", NORM_SHAPES)
@pytest.mark.parametrize("wide", [False, True])
def test_norm_gradients_of_many_rows(dtype, rows, columns, wide):
    gen = torch.Generator(device="cuda").manual_seed(columns + 1)
    x, r, dy, ds = (torch.randn(rows, columns, generator=gen, device="cuda", dtype=torch.float32).to(dtype) for _ in range(4))
    if wide:
        r, ds = r.float(), ds.float()
    weight = torch.randn(columns, generator=gen, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, weight, r)]
    out = ops.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    dx, dweight, dr = torch.autograd.grad(out, leaves, [dy, ds])
    s, g, w = x.double() + r.double(), dy.double(), weight.double()
    rstd = torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6)
    u, du = s * rstd, g * w
    want = rstd * (du - u * (du * u).mean(1, keepdim=True)) + ds.double()
    assert excess(dr, want, r.dtype, 4 * 24 + 24) <= 0
    assert excess(dx, want, dtype, 4 * 24 + 24) <= 0
    # sums over rows of dy u: each term is off by its own error, the sum by one rounding for each of its terms' sizes
    size = (g * u).abs().sum(0)
    want = (g * u).sum(0)
    assert excess(dweight, want, torch.float32, 24, (rows / 16 + 64) * 2.0**-24 * size) <= 0


# ---------------------------------------------------------------------------
# convolution: chunks of many rows, so that rows are refilled and the backward pass's short way is taken


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4])
@pytest.mark.parametrize("batch,length,channels,ends", [(8, 1500, 1024, None), (8, 1500, 1023, [1500, 0, 1, 2, 3, 777, 1024, 1499])])
def test_conv_of_long_chunks(dtype, width, batch, length, channels, ends):
    gen = torch.Generator(device="cuda").manual_seed(width)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, dy = (rand(batch, length, channels).to(dtype) for _ in range(2))
    state, ds = (rand(batch, width - 1, channels).to(dtype) for _ in range(2))
    weight, bias = rand(channels, width), rand(channels)
    lengths = None if ends is None else torch.tensor(ends, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias, state)]
    y, new = ops.causal_conv1d(*leaves[:3], activation="silu", state=leaves[3], lengths=lengths, return_state=True)
    outputs, seeds = ((y, new), (dy, ds)) if width > 1 else ((y,), (dy,))
    dx, dweight, dbias, dstate = torch.autograd.grad(outputs, leaves, seeds, allow_unused=True)

    wide = [t.detach().double().requires_grad_() for t in (x, weight, bias, state)]
    stops = torch.full((batch,), length, device="cuda") if lengths is None else lengths
    live = (torch.arange(length, device="cuda") < stops[:, None])[..., None]
    full = torch.cat([wide[3], wide[0]], 1)
    pre = wide[2].expand(batch, length, channels)
    for j in range(width):
        pre = pre + wide[1][:, j] * full[:, j : j + length]
    want = torch.where(live, torch.nn.functional.silu(pre), 0.0)
    rows = stops[:, None] + torch.arange(width - 1, device="cuda")
    last = full.gather(1, rows[..., None].expand(-1, -1, channels))
    wanted = torch.autograd.grad((want, last) if width > 1 else (want,), wide, [t.double() for t in seeds], allow_unused=True)
    assert excess(y, want.detach(), dtype, width) <= 0
    if width > 1:
        assert torch.equal(new.double(), last.detach())
        assert excess(dstate, wanted[3], dtype, 4 * (width + 8)) <= 0
    assert excess(dx, wanted[0], dtype, 4 * (width + 8)) <= 0
    # the parameters' gradients: sums of batch * length terms, each off by its own exponential's error, a rounding per addition
    # of a chunk's (at most 256) and of the chunks' sums (at most 64 in a row)
    with torch.no_grad():
        gate = torch.sigmoid(pre)
        dpre = (dy.double() * live * gate * (1 + pre * (1 - gate))).abs()
        for got, need, terms in [(dbias, wanted[2], dpre),
                                 *((dweight[:, j], wanted[1][:, j], dpre * full[:, j : j + length].abs()) for j in range(width))]:
            assert excess(got, need, torch.float32, 8, (2.0**-20 + (256 + 64) * 2.0**-24) * terms.sum((0, 1))) <= 0


# ---------------------------------------------------------------------------
# 4-bit products: more units of work than warps


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize(
    "rows,inputs,outputs,group,parts",
    [(1, 4096, 40000, 128, False), (64, 1024, 70003, 64, False), (16, 8192, 16384, 128, True), (64, 4096, 4096, 64, True), (5, 8992, 40000, 32, True)],
)
def test_int4_of_many_units(kind, rows, inputs, outputs, group, parts, zeros):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    packed = torch.randint(0, 256, (outputs, inputs // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = 0.5 + torch.rand(outputs, inputs // group, generator=gen, device="cuda")
    zero = torch.randint(0, 16, (outputs, inputs // group), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    x = torch.randn(rows, inputs, generator=gen, device="cuda")
    x = (x * 40).clamp(-127, 127).to(kind) if kind == torch.int8 else x.to(kind)
    x_scale = 0.5 + torch.rand(rows, generator=gen, device="cuda") if kind in (torch.int8, torch.float8_e4m3fn) else None
    code = {**sequence._DTYPES, **sequence._QUANTIZED}[kind]
    # k in one part or in several; by either plan these outputs are more than one tile of sixteen to a warp
    assert (_lib.load().xe_int4_linear_workspace_size(rows, inputs, outputs, code) > 0) == parts
    y = ops.int4_linear(x, packed, scales, zero, x_scale=x_scale, dtype=torch.float32)
    w = torch.stack([packed & 15, packed >> 4], 2).reshape(outputs, -1, group).double()
    w -= 8.0 if zero is None else zero.double()[..., None]
    w = (w * scales.double()[..., None]).reshape(outputs, inputs)
    xs = x.float().double() * (1.0 if x_scale is None else x_scale.double()[:, None])
    want, size = xs @ w.t(), xs.abs() @ w.t().abs()
    room = (inputs / 16 + 8) * 2.0**-23 * size + 2.0**-24 * want.abs()
    assert ((y.double() - want).abs() <= room).all()


# ---------------------------------------------------------------------------
# scan: lengths run in segments, in every layout of the kernels


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("states", [5, 24, 64])
@pytest.mark.parametrize("groups", [1, 2])
def test_scan_of_a_split_length_in_a_batch(dtype, states, groups):
    """Three sequences that end in different segments, one of them before its first token; last states and all gradients."""
    batch, length, channels = 3, 400, 40
    assert _lib.load().xe_selective_scan_workspace_size(batch, length, channels, states, groups) > 0
    v = scan_inputs(71 + states, batch, length, channels, states, groups, dtype)
    names = list(v)
    gen = torch.Generator().manual_seed(72)
    dy, dstate = randn(gen, batch, length, channels, dtype=dtype), randn(gen, batch, channels, states)
    ends = torch.tensor([0, 130, length])
    w = leaf({k: wide(t) for k, t in v.items()}, names)
    out = scan_reference(w, True, ends)
    want = grads_of(out, [wide(dy), wide(dstate)], [w[k] for k in names])
    for k in ("x", "delta", "b", "c", "z"):
        for i, end in enumerate(ends.tolist()):
            v[k][i, end:] = float("nan")
    g = leaf({k: cuda(t) for k, t in v.items()}, names)
    y, state = scan_call(g, True, ends.cuda(), return_state=True)
    close(y.detach(), out[0].detach(), length)
    close(state.detach(), out[1].detach(), length)
    seed = dy.clone()
    for i, end in enumerate(ends.tolist()):
        seed[i, end:] = float("nan")
    got = grads_of((y, state), [cuda(seed), cuda(dstate)], [g[k] for k in names])
    for k, a, b in zip(names, got, want):
        close(a, b, length + (channels if k in "bc" else batch), factor=4.0)


@pytest.mark.parametrize("batch,length,channels", [(3, 70, 4000), (40, 33, 260)])
def test_scan_of_many_channels(batch, length, channels):
    """Sequences that are not split, of enough channels to fill the device."""
    assert _lib.load().xe_selective_scan_workspace_size(batch, length, channels, 16, 1) == 0
    v = scan_inputs(73, batch, length, channels, 16, 1, torch.bfloat16)
    y, state = scan_call({k: cuda(t) for k, t in v.items()}, True, return_state=True)
    want_y, want_state = scan_reference(v, True)
    close(y, want_y, length)
    close(state, want_state, length)
