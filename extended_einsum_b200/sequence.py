"""Operators along an ordered axis and their quantised projections (the sequence part of ``ops``).

A norm, a projection, a short causal convolution and a selective state space scan: the parts of a layer
that carries a state from token to token.  In the expression graph such a recurrence is a chain
of one einsum per token (interface/tensor_expression.py:196-265); here the whole chain is one call.

Layouts are channel-last: (batch, length, channels).  Inputs may be float32, bfloat16 or float16
with any batch and token strides (the channels are copied together if they are not contiguous);
parameters, statistics and states of the scan are float32; outputs are contiguous.  Every function
checks its arguments, allocates its outputs with torch's caching allocator and launches on torch's
current stream, like the rest of ``ops``.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib

_DTYPES = {torch.float32: _lib.XE_F32, torch.bfloat16: _lib.XE_BF16, torch.float16: _lib.XE_F16}
_QUANTIZED = {torch.float8_e4m3fn: _lib.XE_E4M3, torch.int8: _lib.XE_I8}
_QUANTIZE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_ACTIVATIONS = {None: 0, "silu": 1}


def _device_of(what: str, x: torch.Tensor) -> torch.device:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected torch.Tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"{what}: the B200 kernels take CUDA tensors, got a tensor on {x.device}")
    return x.device


def _dtype_code(what: str, x: torch.Tensor) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise NotImplementedError(f"{what}: float32, bfloat16 and float16 are implemented, got {x.dtype}")
    return code


def _operand(what: str, name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple, dtype: torch.dtype) -> torch.Tensor:
    """Checks one operand and makes its last axis contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected torch.Tensor for {name}, got {type(t).__name__}")
    if t.get_device() != like.get_device():
        raise ValueError(f"{what}: tensors on different devices ({like.device} and {t.device})")
    if t.dtype != dtype:
        raise NotImplementedError(f"{what}: {name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _parameter(what: str, name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple) -> torch.Tensor:
    return _operand(what, name, t, like, shape, torch.float32).contiguous()


def _lengths(what: str, lengths: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor | None:
    if lengths is None:
        return None
    dtype = torch.int64 if lengths.dtype == torch.int64 else torch.int32
    return _operand(what, "lengths", lengths, like, like.shape[:1], dtype).contiguous()


def _pointer(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_entries: dict[str, object] = {}


def _entry(name: str):
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = getattr(_lib.load(), name)
    return entry


def _call(device: torch.device, name: str, *args) -> None:
    """Calls an entry point on the device's current stream (its last argument)."""
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _call(device, name, *args)
    status = _entry(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def _like(x: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """An empty contiguous tensor of x's shape (empty_like alone would keep the order of x's axes)."""
    if x.is_contiguous():
        return torch.empty_like(x, dtype=dtype) if dtype else torch.empty_like(x)
    return torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)


def _needs_grad(what: str, *tensors: torch.Tensor | None) -> bool:
    """Whether autograd records this call.  A forward-mode tangent is refused: it would be dropped."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: no forward-mode derivative")
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return True
    return False


def _no_backward(what: str, *tensors: torch.Tensor | None) -> None:
    if _needs_grad(what, *tensors):
        raise NotImplementedError(f"{what}: no backward pass on this path")


def _workspace(size: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(size, device=device, dtype=torch.uint8) if size else None


# ---------------------------------------------------------------------------
# causal convolution


def causal_conv1d(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    state: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    return_state: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """y[b,t,c] = act(bias[c] + sum_j weight[c,j] v[b,t-width+1+j,c]) (xe_causal_conv1d).

    ``x`` is (batch, length, channels), ``weight`` (channels, width) with width 1 to 4, ``activation``
    None or 'silu'.  ``v`` is x with ``state`` (batch, width - 1, channels; zeros if None) before it;
    ``return_state`` also returns the state after the last token, for a later call or
    ``causal_conv1d_step``.  ``lengths`` (batch,) int32 or int64: only the first so many tokens of
    each sequence count, y is zero after them.  Differentiable (autograd.CausalConv1d).
    """
    if _needs_grad("causal_conv1d", x, weight, bias, state):
        from .autograd import CausalConv1d

        return CausalConv1d.apply(x, weight, bias, state, activation, lengths, return_state)
    y, new = _conv_forward(x, weight, bias, activation, state, lengths, return_state)
    return (y, new) if return_state else y


def _conv_forward(x, weight, bias, activation, state, lengths, return_state):
    x, weight, bias, state, lengths, code = _conv_operands("causal_conv1d", x, weight, bias, state, lengths, activation)
    batch, length, channels = x.shape
    width = weight.shape[1]
    y = _like(x)
    new = torch.empty((batch, width - 1, channels), device=x.device, dtype=x.dtype) if return_state else None
    _call(
        x.device, "xe_causal_conv1d", x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _pointer(bias),
        _pointer(state), y.data_ptr(), _pointer(new), _pointer(lengths), int(lengths is not None and lengths.dtype == torch.int64),
        batch, length, channels, width, _ACTIVATIONS[activation], code,
    )
    return y, new


def _conv_operands(what, x, weight, bias, state, lengths, activation):
    _device_of(what, x)
    code = _dtype_code(what, x)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be (batch, length, channels)")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError(f"{what}: weight must be (channels, width)")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {activation!r}; expected None or 'silu'")
    batch, _, channels = x.shape
    x = _operand(what, "x", x, x, x.shape, x.dtype)
    weight = _parameter(what, "weight", weight, x, (channels, weight.shape[1]))
    if bias is not None:
        bias = _parameter(what, "bias", bias, x, (channels,))
    if state is not None:
        state = _operand(what, "state", state, x, (batch, weight.shape[1] - 1, channels), x.dtype).contiguous()
    return x, weight, bias, state, _lengths(what, lengths, x), code


def causal_conv1d_step(
    state: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
) -> torch.Tensor:
    """One token of ``causal_conv1d`` (xe_causal_conv1d_step): x and y are (batch, channels).

    ``state`` (batch, width - 1, channels), contiguous, is read and shifted in place.
    """
    what = "causal_conv1d_step"
    _no_backward(what, state, x, weight, bias)
    _device_of(what, x)
    code = _dtype_code(what, x)
    if x.dim() != 2 or not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError(f"{what}: x must be (batch, channels) and weight (channels, width)")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {activation!r}; expected None or 'silu'")
    batch, channels = x.shape
    width = weight.shape[1]
    x = _operand(what, "x", x, x, x.shape, x.dtype)
    weight = _parameter(what, "weight", weight, x, (channels, width))
    if bias is not None:
        bias = _parameter(what, "bias", bias, x, (channels,))
    _operand(what, "state", state, x, (batch, width - 1, channels), x.dtype)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state is updated in place and must be contiguous")
    y = _like(x)
    _call(
        x.device, "xe_causal_conv1d_step", x.data_ptr(), x.stride(0), weight.data_ptr(), _pointer(bias), state.data_ptr(),
        y.data_ptr(), batch, channels, width, _ACTIVATIONS[activation], code,
    )
    increment_version(state)
    return y


def causal_conv1d_backward(x, weight, bias, state, activation, lengths, dy, dstate_out, need_dstate):
    """(dx, dweight, dbias, dstate) of ``causal_conv1d`` (xe_causal_conv1d_backward)."""
    what = "causal_conv1d_backward"
    x, weight, bias, state, lengths, code = _conv_operands(what, x, weight, bias, state, lengths, activation)
    batch, length, channels = x.shape
    width = weight.shape[1]
    dx = _like(x)
    dstate = torch.empty((batch, width - 1, channels), device=x.device, dtype=x.dtype) if need_dstate else None
    if batch == 0 or channels == 0:
        return dx, torch.zeros_like(weight), torch.zeros(channels, device=x.device), dstate
    dy = _operand(what, "dy", dy, x, x.shape, x.dtype)
    if dstate_out is not None:
        dstate_out = _operand(what, "the state's gradient", dstate_out, x, (batch, width - 1, channels), x.dtype).contiguous()
    dweight = torch.empty((width + 1, channels), device=x.device, dtype=torch.float32)
    size = _entry("xe_causal_conv1d_backward_workspace_size")(batch, length, channels, width)
    workspace = _workspace(size, x.device)
    _call(
        x.device, "xe_causal_conv1d_backward", x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _pointer(bias),
        _pointer(state), dy.data_ptr(), dy.stride(0), dy.stride(1), _pointer(dstate_out), dx.data_ptr(), _pointer(dstate),
        dweight.data_ptr(), _pointer(lengths), int(lengths is not None and lengths.dtype == torch.int64), batch, length,
        channels, width, _ACTIVATIONS[activation], code, _pointer(workspace), size,
    )
    return dx, dweight[:width].t(), dweight[width], dstate


# ---------------------------------------------------------------------------
# selective scan


def selective_scan(
    x: torch.Tensor,
    delta: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    c: torch.Tensor,
    d: torch.Tensor | None = None,
    *,
    z: torch.Tensor | None = None,
    delta_bias: torch.Tensor | None = None,
    softplus: bool = False,
    state: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    return_state: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """The selective state space scan (xe_selective_scan): for channel d and state n

        dt = delta + delta_bias (then softplus, if set),
        h_t = exp(dt a) h_{t-1} + dt b_t x_t,   y_t = (sum_n c_t h_t + d x_t) * silu(z_t).

    ``x``, ``delta``, ``z`` are (batch, length, channels); ``a`` (channels, states) with at most 64
    states, ``d``, ``delta_bias`` (channels,), float32; ``b``, ``c`` (batch, length, states), or
    (batch, length, groups, states) where groups divide the channels.  ``state`` (batch, channels,
    states), float32, is h before the first token (zero if None); ``return_state`` also returns h after
    the last.  ``lengths`` (batch,): tokens past a sequence's length leave its state alone and give
    y = 0.  Differentiable in every floating operand (autograd.SelectiveScan).
    """
    if _needs_grad("selective_scan", x, delta, a, b, c, d, z, delta_bias, state):
        from .autograd import SelectiveScan

        return SelectiveScan.apply(x, delta, a, b, c, d, z, delta_bias, state, softplus, lengths, return_state)
    y, new, _ = _scan_forward(x, delta, a, b, c, d, z, delta_bias, softplus, state, lengths, return_state, False)
    return (y, new) if return_state else y


def _scan_args(what, x, delta, a, b, c, d, z, delta_bias, softplus, state, lengths):
    """The checked operands as an argument block, and the tensors that it points into."""
    _device_of(what, x)
    code = _dtype_code(what, x)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be (batch, length, channels)")
    if not isinstance(a, torch.Tensor) or a.dim() != 2:
        raise ValueError(f"{what}: a must be (channels, states)")
    batch, length, channels = x.shape
    states = a.shape[1]
    dtype = x.dtype
    x = _operand(what, "x", x, x, x.shape, dtype)
    delta = _operand(what, "delta", delta, x, x.shape, dtype)
    a = _parameter(what, "a", a, x, (channels, states))
    if b.dim() == 3:
        b = b.unsqueeze(2)
    if c.dim() == 3:
        c = c.unsqueeze(2)
    groups = b.shape[2] if b.dim() == 4 else 1
    if groups < 1 or channels % groups:
        raise ValueError(f"{what}: {channels} channels do not divide into {groups} groups")
    b = _operand(what, "b", b, x, (batch, length, groups, states), dtype)
    c = _operand(what, "c", c, x, (batch, length, groups, states), dtype)
    if d is not None:
        d = _parameter(what, "d", d, x, (channels,))
    if z is not None:
        z = _operand(what, "z", z, x, x.shape, dtype)
    if delta_bias is not None:
        delta_bias = _parameter(what, "delta_bias", delta_bias, x, (channels,))
    if state is not None:
        state = _parameter(what, "state", state, x, (batch, channels, states))
    lengths = _lengths(what, lengths, x)
    zb, zt = (z.stride(0), z.stride(1)) if z is not None else (0, 0)
    args = _lib.SelectiveScanArgs(
        x.data_ptr(), delta.data_ptr(), _pointer(z), b.data_ptr(), c.data_ptr(), None, a.data_ptr(), _pointer(d),
        _pointer(delta_bias), _pointer(state), None, None, _pointer(lengths),
        x.stride(0), x.stride(1), delta.stride(0), delta.stride(1), zb, zt,
        b.stride(0), b.stride(1), b.stride(2), c.stride(0), c.stride(1), c.stride(2),
        batch, length, channels, states, groups,
        int(lengths is not None and lengths.dtype == torch.int64), int(softplus), code,
    )
    return args, (x, delta, z, b, c, a, d, delta_bias, state, lengths), groups


def _scan_forward(x, delta, a, b, c, d, z, delta_bias, softplus, state, lengths, return_state, training):
    what = "selective_scan"
    args, kept, groups = _scan_args(what, x, delta, a, b, c, d, z, delta_bias, softplus, state, lengths)
    x = kept[0]
    batch, length, channels = x.shape
    states = a.shape[1]
    y = _like(x)
    args.y = y.data_ptr()
    new = checkpoints = None
    if return_state:
        new = torch.empty((batch, channels, states), device=x.device, dtype=torch.float32)
        args.state_out = new.data_ptr()
    if training:
        size = _entry("xe_selective_scan_checkpoint_size")(batch, length, channels, states)
        checkpoints = torch.empty(size // 4, device=x.device, dtype=torch.float32)
        args.checkpoints = checkpoints.data_ptr()
    size = _entry("xe_selective_scan_workspace_size")(batch, length, channels, states, groups)
    workspace = _workspace(size, x.device)
    _call(x.device, "xe_selective_scan", args, _pointer(workspace), size)
    return y, new, checkpoints


def selective_scan_step(
    state: torch.Tensor,
    x: torch.Tensor,
    delta: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    c: torch.Tensor,
    d: torch.Tensor | None = None,
    *,
    z: torch.Tensor | None = None,
    delta_bias: torch.Tensor | None = None,
    softplus: bool = False,
) -> torch.Tensor:
    """One token of ``selective_scan`` (xe_selective_scan_step): x, delta, z and y are (batch, channels),
    b and c (batch, states) or (batch, groups, states).  ``state`` (batch, channels, states), float32 and
    contiguous, is read and overwritten in place.
    """
    what = "selective_scan_step"
    _no_backward(what, state, x, delta, a, b, c, d, z, delta_bias)
    _device_of(what, x)
    code = _dtype_code(what, x)
    if x.dim() != 2 or not isinstance(a, torch.Tensor) or a.dim() != 2:
        raise ValueError(f"{what}: x must be (batch, channels) and a (channels, states)")
    batch, channels = x.shape
    states = a.shape[1]
    dtype, shape = x.dtype, x.shape
    x = _operand(what, "x", x, x, shape, dtype)
    delta = _operand(what, "delta", delta, x, shape, dtype)
    a = _parameter(what, "a", a, x, (channels, states))
    if b.dim() == 2:
        b = b.unsqueeze(1)
    if c.dim() == 2:
        c = c.unsqueeze(1)
    groups = b.shape[1] if b.dim() == 3 else 1
    if groups < 1 or channels % groups:
        raise ValueError(f"{what}: {channels} channels do not divide into {groups} groups")
    b = _operand(what, "b", b, x, (batch, groups, states), dtype)
    c = _operand(what, "c", c, x, (batch, groups, states), dtype)
    if d is not None:
        d = _parameter(what, "d", d, x, (channels,))
    if z is not None:
        z = _operand(what, "z", z, x, shape, dtype)
    if delta_bias is not None:
        delta_bias = _parameter(what, "delta_bias", delta_bias, x, (channels,))
    _operand(what, "state", state, x, (batch, channels, states), torch.float32)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state is updated in place and must be contiguous")
    y = _like(x)
    args = _lib.SelectiveScanArgs(
        x.data_ptr(), delta.data_ptr(), _pointer(z), b.data_ptr(), c.data_ptr(), y.data_ptr(), a.data_ptr(), _pointer(d),
        _pointer(delta_bias), None, state.data_ptr(), None, None,
        x.stride(0), 0, delta.stride(0), 0, z.stride(0) if z is not None else 0, 0,
        b.stride(0), 0, b.stride(1), c.stride(0), 0, c.stride(1),
        batch, 1, channels, states, groups, 0, int(softplus), code,
    )
    _call(x.device, "xe_selective_scan_step", args)
    increment_version(state)
    return y


def selective_scan_backward(x, delta, a, b, c, d, z, delta_bias, softplus, state, lengths, checkpoints, dy, dstate_out):
    """Gradients of ``selective_scan`` as a dict (xe_selective_scan_backward), from the forward call's checkpoints."""
    what = "selective_scan_backward"
    args, kept, groups = _scan_args(what, x, delta, a, b, c, d, z, delta_bias, softplus, state, lengths)
    x = kept[0]
    batch, length, channels = x.shape
    states = a.shape[1]
    device, dtype = x.device, x.dtype

    dx, ddelta, dz = _like(x), _like(x), _like(x) if z is not None else None
    db, dc = (torch.empty((batch, length, groups, states), device=device, dtype=dtype) for _ in range(2))
    da = torch.empty((channels, states), device=device, dtype=torch.float32)
    dd = torch.empty((2, channels), device=device, dtype=torch.float32)
    dstate = torch.empty((batch, channels, states), device=device, dtype=torch.float32) if state is not None else None
    if batch and channels:
        dy = _operand(what, "dy", dy, x, x.shape, dtype)
        if dstate_out is not None:
            dstate_out = _parameter(what, "the state's gradient", dstate_out, x, (batch, channels, states))
        args.checkpoints = checkpoints.data_ptr()
        grads = _lib.SelectiveScanGrads(
            dy.data_ptr(), _pointer(dstate_out), dx.data_ptr(), ddelta.data_ptr(), _pointer(dz), db.data_ptr(),
            dc.data_ptr(), da.data_ptr(), dd.data_ptr(), _pointer(dstate), dy.stride(0), dy.stride(1),
        )
        size = _entry("xe_selective_scan_backward_workspace_size")(batch, length, channels, states, groups)
        workspace = _workspace(size, device)
        _call(device, "xe_selective_scan_backward", args, grads, _pointer(workspace), size)
    else:
        da.zero_(), dd.zero_(), db.zero_(), dc.zero_()
    return {"x": dx, "delta": ddelta, "a": da, "b": db.view(b.shape), "c": dc.view(c.shape), "d": dd[0], "z": dz,
            "delta_bias": dd[1], "state": dstate}


# ---------------------------------------------------------------------------
# norm


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    *,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    quantize: str | None = None,
):
    """y = s * rsqrt(mean(s^2) + eps) * weight over the last axis, s = x + residual (xe_rms_norm).

    ``residual`` (x's shape; x's type or float32) and ``weight`` (last axis; x's type or float32) may be
    None.  ``quantize`` 'e4m3' or 'int8' gives y as 8-bit values and one float32 scale per row,
    y ~ q * scale with scale = max(max|y| / (448 or 127), 2^-126): the (values, scale) pair that
    ``int4_linear`` takes.  Returns y, or (q, scale), followed by s (of the residual's type) if there is a
    residual: y; (y, s); (q, scale); (q, scale, s).  Differentiable without ``quantize``
    (autograd.RmsNorm).
    """
    what = "rms_norm"
    if _needs_grad(what, x, weight, residual):
        if quantize is not None:
            raise NotImplementedError(f"{what}: no backward pass through 8-bit outputs")
        from .autograd import RmsNorm

        return RmsNorm.apply(x, weight, residual, eps)
    return _norm_forward(x, weight, residual, eps, quantize)


def _norm_forward(x, weight, residual, eps, quantize):
    what = "rms_norm"
    device = _device_of(what, x)
    code = _dtype_code(what, x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what}: needs a last axis of at least one element")
    rows = _as_rows(x)
    count, columns = rows.shape
    weight_ptr = residual_ptr = sum_ptr = scale_ptr = None
    weight_code, residual_code, residual_row = _lib.XE_F32, code, 0
    if weight is not None:
        if weight.dtype != torch.float32:
            weight_code = code
        weight = _operand(what, "weight", weight, x, (columns,), torch.float32 if weight_code == _lib.XE_F32 else x.dtype)
        weight = weight.contiguous()
        weight_ptr = weight.data_ptr()
    total = scale = None
    if residual is not None:
        if residual.dtype == torch.float32:
            residual_code = _lib.XE_F32
        residual = _as_rows(_operand(what, "residual", residual, x, x.shape, torch.float32 if residual_code == _lib.XE_F32 else x.dtype))
        total = _like(x, residual.dtype)
        residual_ptr, residual_row, sum_ptr = residual.data_ptr(), residual.stride(0), total.data_ptr()
    if quantize is None:
        y, out_code = _like(x), code
    elif quantize in _QUANTIZE:
        y = _like(x, _QUANTIZE[quantize])
        out_code = _QUANTIZED[y.dtype]
        scale = torch.empty(x.shape[:-1], device=device, dtype=torch.float32)
        scale_ptr = scale.data_ptr()
    else:
        raise ValueError(f"{what}: unknown quantize {quantize!r}; expected None, 'e4m3' or 'int8'")
    _call(
        device, "xe_rms_norm", rows.data_ptr(), rows.stride(0), residual_ptr, residual_row, weight_ptr, y.data_ptr(),
        sum_ptr, scale_ptr, count, columns, eps, code, residual_code, weight_code, out_code,
    )
    if scale is None:
        return y if total is None else (y, total)
    return (y, scale) if total is None else (y, scale, total)


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, columns) with contiguous columns; a copy only where the rows have no common stride."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def rms_norm_backward(total, addend, weight, dy, dtotal, eps, need_dweight):
    """(dx, dweight) of the norm of total, or total + addend (xe_rms_norm_backward); dx has total's type and shape."""
    what = "rms_norm_backward"
    device = _device_of(what, total)
    code = _dtype_code(what, dy)
    wide = total.dtype == torch.float32
    sum_code = _lib.XE_F32 if wide else code
    weight_code = _lib.XE_F32 if weight is None or weight.dtype == torch.float32 else code
    rows, dy_rows = _as_rows(total), _as_rows(dy)
    if addend is not None:
        addend = _as_rows(addend)
    dsum = None if dtotal is None else _as_rows(_operand(what, "the sum's gradient", dtotal, total, total.shape, total.dtype))
    dx = _like(total)
    columns = total.shape[-1]
    dweight = torch.empty(columns, device=device, dtype=torch.float32) if need_dweight else None
    if rows.shape[0] == 0:
        return dx, None if dweight is None else dweight.zero_()
    if weight is not None:
        weight = weight.contiguous()
    size = _entry("xe_rms_norm_backward_workspace_size")(rows.shape[0], columns) if need_dweight else 0
    workspace = _workspace(size, device)
    _call(
        device, "xe_rms_norm_backward", rows.data_ptr(), rows.stride(0), _pointer(addend),
        0 if addend is None else addend.stride(0), _pointer(weight), dy_rows.data_ptr(), dy_rows.stride(0), _pointer(dsum), 0 if dsum is None else dsum.stride(0), dx.data_ptr(), _pointer(dweight), rows.shape[0],
        columns, eps, code, sum_code, weight_code, _pointer(workspace), size,
    )
    return dx, dweight


# ---------------------------------------------------------------------------
# 4-bit weights


def int4_linear(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    zeros: torch.Tensor | None = None,
    *,
    x_scale: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """y[..., o] = sum_k x[..., k] scales[o, k // group] (q[o, k] - zeros[o, k // group]) (xe_int4_linear).

    ``packed`` (outputs, inputs / 2) uint8 holds two codes to a byte, the even k in the low nibble
    (``int4_pack``); ``scales`` (outputs, inputs / group) float32, bfloat16 or float16 and ``zeros`` uint8 of
    the same shape, 0 to 15 as the codes are (None: 8); the group is a multiple of 32.  ``x`` (..., inputs) is float32, bfloat16 or
    float16, or 8-bit (float8_e4m3fn, int8) with ``x_scale`` (...) as ``rms_norm`` gives them.  ``dtype`` of
    the result: x's type, or bfloat16 for 8-bit x, unless given.  Integers q - zero and the activations
    multiply exactly; sums and scales are float32.  Made for the few rows of token-by-token generation;
    many rows go in slices that share a workspace of at most 512 MB.
    """
    what = "int4_linear"
    _no_backward(what, x, scales, x_scale)
    device = _device_of(what, x)
    code = _DTYPES.get(x.dtype)
    if code is None:
        code = _QUANTIZED.get(x.dtype)
        if code is None:
            raise NotImplementedError(f"{what}: x of {x.dtype} is not implemented")
        if dtype is None:
            dtype = torch.bfloat16
    elif x_scale is not None:
        raise ValueError(f"{what}: x_scale belongs to 8-bit x, got {x.dtype}")
    if dtype is None:
        dtype = x.dtype
    y_code = _DTYPES.get(dtype)
    if y_code is None:
        raise NotImplementedError(f"{what}: a result of {dtype} is not implemented")
    if x.dim() == 0 or packed.dim() != 2 or scales.dim() != 2:
        raise ValueError(f"{what}: expected x (..., inputs), packed (outputs, inputs / 2), scales (outputs, groups)")
    inputs, (outputs, groups) = x.shape[-1], scales.shape
    if inputs == 0 or inputs % 2 or groups == 0 or inputs % groups:
        raise ValueError(f"{what}: {inputs} inputs do not divide into {groups} groups")
    packed = _operand(what, "packed", packed, x, (outputs, inputs // 2), torch.uint8)
    if packed.stride(0) % 16 or packed.data_ptr() % 16:
        packed = packed.clone(memory_format=torch.contiguous_format)
    scale_code = _DTYPES.get(scales.dtype)
    if scale_code is None:
        raise NotImplementedError(f"{what}: scales of {scales.dtype} are not implemented")
    scales = _operand(what, "scales", scales, x, (outputs, groups), scales.dtype).contiguous()
    if zeros is not None:
        zeros = _operand(what, "zeros", zeros, x, (outputs, groups), torch.uint8).contiguous()
    rows = _as_rows(x)
    if x_scale is not None:
        x_scale = _operand(what, "x_scale", x_scale, x, x.shape[:-1], torch.float32).contiguous()
    y = torch.empty((*x.shape[:-1], outputs), device=device, dtype=dtype)
    size = _entry("xe_int4_linear_workspace_size")(rows.shape[0], inputs, outputs, code)
    workspace = _workspace(size, device)
    _call(
        device, "xe_int4_linear", rows.data_ptr(), rows.stride(0), _pointer(x_scale), packed.data_ptr(), packed.stride(0),
        scales.data_ptr(), _pointer(zeros), y.data_ptr(), rows.shape[0], inputs, outputs, inputs // groups, code, scale_code,
        y_code, _pointer(workspace), size,
    )
    return y


def int4_pack(codes: torch.Tensor) -> torch.Tensor:
    """Codes 0 to 15, (outputs, inputs), two to a byte with the even input in the low nibble."""
    if codes.dim() != 2 or codes.shape[1] % 2:
        raise ValueError("int4_pack: expected (outputs, inputs) with an even number of inputs")
    if ((codes < 0) | (codes > 15)).any():
        raise ValueError("int4_pack: codes are whole numbers from 0 to 15")
    codes = codes.to(torch.uint8)
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def int4_quantize(
    weight: torch.Tensor, group: int = 128, *, symmetric: bool = True, scale_dtype: torch.dtype | None = None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """(packed, scales, zeros) of a (outputs, inputs) weight, once when it is loaded: each group's values round to
    the nearest of 16 levels, -7 .. 7 times the scale (``symmetric``; zeros None), or levels from its minimum to
    its maximum, zero among them, with a whole zero point.  The scales are rounded to ``scale_dtype`` (the weight's
    type) before the codes are taken."""
    if weight.dim() != 2 or group < 32 or group % 32 or weight.shape[1] % group:
        raise ValueError(f"int4_quantize: shape {tuple(weight.shape)} in groups of {group} (a multiple of 32)")
    scale_dtype = scale_dtype or weight.dtype
    if scale_dtype not in _DTYPES:
        raise NotImplementedError(f"int4_quantize: scales of {scale_dtype} are not implemented")
    w = weight.float().reshape(weight.shape[0], -1, group)
    if symmetric:
        scales, zeros = (w.abs().amax(2) / 7.0), None
    else:
        low, high = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
        scales = (high - low) / 15.0
    tiny = torch.finfo(scale_dtype).tiny
    scales = scales.clamp(min=tiny).to(scale_dtype)
    step = scales.float()
    if symmetric:
        codes = torch.round(w / step[:, :, None]).clamp(-8, 7) + 8.0
    else:
        zero = torch.round(-low / step).clamp(0, 15)
        zeros = zero.to(torch.uint8)
        codes = (torch.round(w / step[:, :, None]) + zero[:, :, None]).clamp(0, 15)
    return int4_pack(codes.reshape(weight.shape)), scales, zeros
