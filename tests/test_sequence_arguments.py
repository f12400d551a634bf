"""What the sequence operators' wrappers hand to their entry points and keep from them (no GPU)."""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import ops, sequence


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
