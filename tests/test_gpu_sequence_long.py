"""The sequence operators at sizes where their kernels run for many turns, against their float64 definitions.

Tolerances as in test_gpu_sequence.py, whose helpers and derivations these are.
"""

from __future__ import annotations

import pytest
import torch

from extended_einsum_b200 import _lib, ops
from test_gpu_sequence import TYPES, cuda, int4_close, int4_inputs, randn

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
