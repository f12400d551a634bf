"""What the sequence operators refuse, and their C entry points' checks (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from extended_einsum_b200 import _lib, ops


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv1d(x, torch.zeros(8, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv1d_step(torch.zeros(2, 3, 8), x[:, 0], torch.zeros(8, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.selective_scan_step(torch.zeros(2, 8, 4), x[:, 0], x[:, 0], torch.zeros(8, 4), torch.zeros(2, 4), torch.zeros(2, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.rms_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int4_linear(x, torch.zeros(3, 4, dtype=torch.uint8), torch.zeros(3, 1))
    with pytest.raises(TypeError):
        ops.rms_norm([1.0, 2.0])


def test_int4_pack_and_quantize_on_the_host():
    codes = torch.arange(64).remainder(16).reshape(2, 32)
    packed = ops.int4_pack(codes)
    assert packed.dtype == torch.uint8 and packed.shape == (2, 16)
    assert torch.equal(packed & 15, codes[:, 0::2].to(torch.uint8)) and torch.equal(packed >> 4, codes[:, 1::2].to(torch.uint8))
    with pytest.raises(ValueError):
        ops.int4_pack(torch.zeros(2, 3))
    with pytest.raises(ValueError):
        ops.int4_quantize(torch.zeros(4, 96), 64)
    with pytest.raises(NotImplementedError):
        ops.int4_quantize(torch.zeros(4, 64), 32, scale_dtype=torch.float64)
    packed, scales, zeros = ops.int4_quantize(torch.zeros(4, 64), 32)  # a zero weight stays zero
    assert zeros is None and (packed == 0x88).all() and (scales > 0).all()


def scan_args(**changes):
    q = _lib.SelectiveScanArgs()
    for name in ("x", "delta", "b", "c", "y", "a"):
        setattr(q, name, 256)
    q.batch, q.length, q.channels, q.states, q.groups, q.dtype = 1, 4, 8, 4, 1, _lib.XE_F32
    for name, value in changes.items():
        setattr(q, name, value)
    return q


@pytest.mark.parametrize(
    "changes,status,message",
    [
        ({"x": None}, _lib.XE_ERR_INVALID_ARGUMENT, "null"),
        ({"a": None}, _lib.XE_ERR_INVALID_ARGUMENT, "null"),
        ({"y": None}, _lib.XE_ERR_INVALID_ARGUMENT, "null"),
        ({"dtype": 9}, _lib.XE_ERR_NOT_SUPPORTED, "type"),
        ({"states": 65}, _lib.XE_ERR_NOT_SUPPORTED, "states"),
        ({"states": 0}, _lib.XE_ERR_INVALID_ARGUMENT, "states"),
        ({"groups": 3}, _lib.XE_ERR_INVALID_ARGUMENT, "groups"),
        ({"batch": -1}, _lib.XE_ERR_INVALID_ARGUMENT, "negative"),
        ({"batch": 70000}, _lib.XE_ERR_NOT_SUPPORTED, "limit"),
    ],
)
def test_scan_entry_refuses(changes, status, message):
    lib = _lib.load()
    assert lib.xe_selective_scan(scan_args(**changes), None, 0, None) == status
    assert message in _lib.last_error()


def test_scan_entries_need_their_buffers():
    lib = _lib.load()
    # a long sequence of few channels is split, and then needs a workspace
    size = lib.xe_selective_scan_workspace_size(1, 4096, 8, 4, 1)
    assert size > 0
    assert lib.xe_selective_scan(scan_args(length=4096), None, 0, None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert "workspace" in _lib.last_error()
    assert lib.xe_selective_scan_step(scan_args(), None) == _lib.XE_ERR_INVALID_ARGUMENT  # no state
    assert lib.xe_selective_scan_backward(scan_args(), None, None, 0, None) == _lib.XE_ERR_INVALID_ARGUMENT
    grads = _lib.SelectiveScanGrads()
    assert lib.xe_selective_scan_backward(scan_args(), grads, None, 0, None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert lib.xe_selective_scan_checkpoint_size(1, 9, 8, 17) == 2 * 8 * 32 * 4
    assert lib.xe_selective_scan(scan_args(batch=0, x=None, y=None), None, 0, None) == _lib.XE_OK


def test_convolution_entry_refuses():
    lib = _lib.load()

    def conv(x=256, weight=256, y=256, batch=1, length=4, channels=8, width=4, activation=1, dtype=0):
        return lib.xe_causal_conv1d(x, 0, 8, weight, None, None, y, None, None, 0, batch, length, channels, width, activation,
                                    dtype, None)

    assert conv(x=None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert conv(weight=None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert conv(width=0) == _lib.XE_ERR_INVALID_ARGUMENT
    assert conv(width=5) == _lib.XE_ERR_NOT_SUPPORTED
    assert conv(activation=2) == _lib.XE_ERR_INVALID_ARGUMENT
    assert conv(dtype=3) == _lib.XE_ERR_NOT_SUPPORTED
    assert conv(length=-1) == _lib.XE_ERR_INVALID_ARGUMENT
    assert conv(x=None, y=None, batch=0) == _lib.XE_OK
    step = lib.xe_causal_conv1d_step(256, 8, 256, None, None, 256, 1, 8, 4, 0, 0, None)
    assert step == _lib.XE_ERR_INVALID_ARGUMENT and "state" in _lib.last_error()
    back = lib.xe_causal_conv1d_backward(256, 0, 8, 256, None, None, 256, 0, 8, None, 256, None, 256, None, 0, 1, 4, 8, 4, 1, 0,
                                         None, 0, None)
    assert back == _lib.XE_ERR_INVALID_ARGUMENT and "workspace" in _lib.last_error()


def test_norm_entry_refuses():
    lib = _lib.load()

    def norm(x=256, residual=None, y=256, total=None, scale=None, rows=2, columns=8, types=(0, 0, 0, 0)):
        return lib.xe_rms_norm(x, 8, residual, 8, None, y, total, scale, rows, columns, ctypes.c_float(1e-6), *types, None)

    assert norm(x=None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert norm(residual=256) == _lib.XE_ERR_INVALID_ARGUMENT  # nowhere to put the sum
    assert norm(columns=0) == _lib.XE_ERR_INVALID_ARGUMENT
    assert norm(columns=65537) == _lib.XE_ERR_NOT_SUPPORTED
    assert norm(types=(0, 1, 0, 0)) == _lib.XE_ERR_NOT_SUPPORTED  # float32 rows on a bfloat16 residual
    assert norm(types=(1, 1, 2, 1)) == _lib.XE_ERR_NOT_SUPPORTED
    assert norm(types=(0, 0, 0, 1)) == _lib.XE_ERR_NOT_SUPPORTED
    assert norm(types=(0, 0, 0, 3)) == _lib.XE_ERR_INVALID_ARGUMENT and "scales" in _lib.last_error()
    assert norm(x=None, y=None, rows=0) == _lib.XE_OK


def test_int4_entry_refuses():
    lib = _lib.load()

    def linear(x=256, packed=256, row=32, rows=1, inputs=64, outputs=4, group=32, types=(1, 1, 1)):
        return lib.xe_int4_linear(x, 64, None, packed, row, 256, None, 256, rows, inputs, outputs, group, *types, None, 0, None)

    assert linear(x=None) == _lib.XE_ERR_INVALID_ARGUMENT
    assert linear(packed=264) == _lib.XE_ERR_INVALID_ARGUMENT and "16-byte" in _lib.last_error()
    assert linear(row=24) == _lib.XE_ERR_INVALID_ARGUMENT
    assert linear(group=48) == _lib.XE_ERR_INVALID_ARGUMENT
    assert linear(group=16) == _lib.XE_ERR_NOT_SUPPORTED
    assert linear(types=(7, 1, 1)) == _lib.XE_ERR_NOT_SUPPORTED
    assert linear(types=(1, 3, 1)) == _lib.XE_ERR_NOT_SUPPORTED
    assert linear(inputs=1 << 21, group=1 << 21) == _lib.XE_ERR_NOT_SUPPORTED
    need = lib.xe_int4_linear_workspace_size(16, 8192, 16384, _lib.XE_E4M3)  # k in parts
    assert need > 0
    assert linear(rows=16, inputs=8192, outputs=16384, group=64) == _lib.XE_ERR_INVALID_ARGUMENT
    assert "workspace" in _lib.last_error()
    assert linear(x=None, rows=0) == _lib.XE_OK
