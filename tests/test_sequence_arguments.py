"""What the sequence operators' wrappers hand to their entry points and keep from them (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from torch.autograd import forward_ad

from extended_einsum_b200 import _lib, ops, sequence


@pytest.fixture
def calls(monkeypatch):
    """The wrappers on CPU tensors, their launches recorded instead of made."""
    made = []
    monkeypatch.setattr(sequence, "_device_of", lambda what, x: x.device)
    monkeypatch.setattr(sequence, "_call", lambda device, name, *args: made.append((name, args)))
    return made


def test_int4_scale_of_a_single_row_is_checked(calls):
    """The scale's address goes to the kernel as that of float32 values, whatever the rank of x."""
    packed, scales = torch.zeros(3, 32, dtype=torch.uint8), torch.ones(3, 2)
    for shape in ((64,), (2, 64)):
        x = torch.zeros(shape, dtype=torch.int8)
        scale = torch.ones(shape[:-1])
        ops.int4_linear(x, packed, scales, x_scale=scale)
        assert calls.pop()[1][2] == scale.data_ptr()
        with pytest.raises(NotImplementedError, match="x_scale"):
            ops.int4_linear(x, packed, scales, x_scale=scale.double())
        with pytest.raises(ValueError, match="x_scale has shape"):
            ops.int4_linear(x, packed, scales, x_scale=torch.ones(5))
        with pytest.raises(TypeError, match="x_scale"):
            ops.int4_linear(x, packed, scales, x_scale=0.5)
    assert not calls


def test_steps_tell_autograd_of_the_state(calls):
    """The state is written through its address: its version moves on, so that a graph that saved it fails and does not use
    what it has become."""
    taps, held = torch.zeros(2, 3, 8), torch.zeros(2, 8, 4)
    x, bc = torch.zeros(2, 8), torch.zeros(2, 4)
    for state, step in (
        (taps, lambda: ops.causal_conv1d_step(taps, x, torch.zeros(8, 4))),
        (held, lambda: ops.selective_scan_step(held, x, x, torch.zeros(8, 4), bc, bc)),
    ):
        before = state._version
        step()
        assert state._version > before and len(calls) == 1
        calls.clear()
        scale = torch.ones((), requires_grad=True)
        out = (state * scale).sum()  # saves the state
        with torch.no_grad():
            step()
        calls.clear()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()
    with torch.inference_mode():  # such tensors have no version
        ops.causal_conv1d_step(torch.zeros(2, 3, 8), x, torch.zeros(8, 4))
        held = torch.zeros(2, 8, 4)
    ops.selective_scan_step(held, x, x, torch.zeros(8, 4), bc, bc)


def test_forward_mode_is_refused():
    """No operator here has a forward-mode derivative: a tangent is refused, not dropped."""
    three, row = torch.zeros(2, 3, 8), torch.zeros(2, 8)
    bc = torch.zeros(2, 3, 4)
    uses = [
        (three, lambda t: ops.causal_conv1d(t, torch.zeros(8, 4))),
        (torch.zeros(8), lambda t: ops.causal_conv1d(three, torch.zeros(8, 4), t)),
        (row, lambda t: ops.causal_conv1d_step(torch.zeros(2, 3, 8), t, torch.zeros(8, 4))),
        (bc, lambda t: ops.selective_scan(three, three, torch.zeros(8, 4), t, bc)),
        (torch.zeros(2, 8, 4), lambda t: ops.selective_scan(three, three, torch.zeros(8, 4), bc, bc, state=t)),
        (row, lambda t: ops.selective_scan_step(torch.zeros(2, 8, 4), row, t, torch.zeros(8, 4), bc[:, 0], bc[:, 0])),
        (three, lambda t: ops.rms_norm(t)),
        (three, lambda t: ops.rms_norm(three, residual=t, quantize="int8")),
        (torch.zeros(2, 64), lambda t: ops.int4_linear(t, torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 1))),
        (torch.zeros(3, 1), lambda t: ops.int4_linear(torch.zeros(2, 64), torch.zeros(3, 32, dtype=torch.uint8), t)),
    ]
    for value, use in uses:
        for grad in (False, True):
            for requires in (False, True):
                primal = value.clone().requires_grad_(requires)
                with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    dual = forward_ad.make_dual(primal, torch.ones_like(value))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        use(dual)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="CUDA"):
        ops.rms_norm(three)  # no tangent: on to the next check


@pytest.mark.parametrize("rows", [16384, 70000, 1 << 20])
@pytest.mark.parametrize("dtype", [_lib.XE_F32, _lib.XE_BF16, _lib.XE_E4M3])
@pytest.mark.parametrize("inputs,outputs", [(4096, 16384), (8192, 16384), (18432, 20)])
def test_int4_workspace_of_many_rows_is_bounded(rows, dtype, inputs, outputs):
    """Prompts go in slices: their partial sums do not grow with the rows without end (6.4 GB for 16384 rows of the second
    shape at once)."""
    lib = _lib.load()
    one = lib.xe_int4_linear_workspace_size(21 if dtype == _lib.XE_F32 else 64, inputs, outputs, dtype)
    assert 0 < one <= lib.xe_int4_linear_workspace_size(rows, inputs, outputs, dtype) <= 512 << 20


def test_int4_entry_takes_many_rows():
    """More rows than a grid holds are no reason to refuse."""
    lib = _lib.load()
    status = lib.xe_int4_linear(256, 64, None, 256, 32, None, None, 256, 70000, 64, 4, 32, 1, 1, 1, None, 0, None)
    assert status == _lib.XE_ERR_INVALID_ARGUMENT and "null" in _lib.last_error()  # no scales: the size has passed
    status = lib.xe_int4_linear(256, 8192, None, 256, 4096, 256, None, 256, 70000, 8192, 20, 32, 1, 1, 1, None, 0, None)
    assert status == _lib.XE_ERR_INVALID_ARGUMENT and "workspace" in _lib.last_error()


def test_entries_refuse_buffers_off_their_boundaries():
    """Workspaces and the stored states are written in vectors: a place that does not allow it is refused, not faulted on."""
    lib = _lib.load()
    q = _lib.SelectiveScanArgs()
    for name in ("x", "delta", "b", "c", "y", "a", "state_out", "checkpoints"):
        setattr(q, name, 4096)
    q.batch, q.length, q.channels, q.states, q.groups, q.dtype = 1, 4096, 8, 4, 1, _lib.XE_F32
    grads = _lib.SelectiveScanGrads(*([4096] * 10), 8, 8)

    def conv(workspace):
        return lib.xe_causal_conv1d_backward(4096, 0, 8, 4096, None, None, 4096, 0, 8, None, 4096, None, 4096, None, 0, 1, 4, 8, 4,
                                             1, 0, workspace, 1 << 30, None)

    def norm(workspace):
        return lib.xe_rms_norm_backward(4096, 8, None, 0, None, 4096, 8, None, 0, 4096, 4096, 2, 8, ctypes.c_float(1e-6), 0, 0, 0,
                                        workspace, 1 << 30, None)

    def int4(workspace):
        return lib.xe_int4_linear(4096, 8192, None, 4096, 4096, 4096, None, 4096, 64, 8192, 64, 32, 1, 1, 1, workspace, 1 << 30, None)

    for call in (conv, norm, int4, lambda w: lib.xe_selective_scan(q, w, 1 << 30, None),
                 lambda w: lib.xe_selective_scan_backward(q, grads, w, 1 << 30, None)):
        for workspace in (4096 + 4, 4096 + 128):
            assert call(workspace) == _lib.XE_ERR_INVALID_ARGUMENT and "aligned" in _lib.last_error()
    q.checkpoints = 4096 + 8
    assert lib.xe_selective_scan(q, 4096, 1 << 30, None) == _lib.XE_ERR_INVALID_ARGUMENT and "aligned" in _lib.last_error()
    assert lib.xe_selective_scan_backward(q, grads, 4096, 1 << 30, None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert "aligned" in _lib.last_error()


@pytest.mark.parametrize("value", [16, 255, 300, -1])
def test_int4_pack_refuses_codes_of_more_than_four_bits(value):
    """They would change their neighbours' codes."""
    codes = torch.full((2, 32), 5)
    codes[1, 3] = value
    with pytest.raises(ValueError, match="0 to 15"):
        ops.int4_pack(codes)
    codes[1, 3] = 15
    assert ops.int4_pack(codes)[1, 1] == 0xF5
    assert ops.int4_pack(codes[:0]).shape == (0, 16)
