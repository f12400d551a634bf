"""The sequence operators in float64 on the CPU, from their definitions: token by token, no shortcuts.

Differentiable by torch, so that gradients follow from the same definitions.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F


def causal_conv1d(x, weight, bias=None, *, activation=None, state=None, lengths=None):
    """(y, new state); x (batch, length, channels), weight (channels, width), state (batch, width - 1, channels)."""
    batch, length, channels = x.shape
    width = weight.shape[1]
    before = state if state is not None else x.new_zeros(batch, width - 1, channels)
    ends = [length] * batch if lengths is None else [min(max(int(n), 0), length) for n in lengths]
    ys, news = [], []
    for i in range(batch):
        v = torch.cat([before[i], x[i, : ends[i]]])
        rows = []
        for t in range(length):
            if t >= ends[i]:
                rows.append(torch.zeros_like(x[i, 0]))
                continue
            y = (v[t : t + width] * weight.t()).sum(0)
            if bias is not None:
                y = y + bias
            rows.append(F.silu(y) if activation == "silu" else y)
        ys.append(torch.stack(rows) if rows else x.new_zeros(0, channels))
        news.append(v[ends[i] : ends[i] + width - 1])
    return torch.stack(ys), torch.stack(news)


def selective_scan(x, delta, a, b, c, d=None, *, z=None, delta_bias=None, softplus=False, state=None, lengths=None):
    """(y, last state); b and c (batch, length, groups, states)."""
    batch, length, channels = x.shape
    each = channels // b.shape[2]
    h = state if state is not None else x.new_zeros(batch, channels, a.shape[1])
    live = None if lengths is None else torch.as_tensor(lengths)
    rows = []
    for t in range(length):
        dt = delta[:, t] + (delta_bias if delta_bias is not None else 0.0)
        if softplus:
            dt = F.softplus(dt, threshold=40.0)
        bt, ct = (v[:, t].repeat_interleave(each, dim=1) for v in (b, c))
        new = torch.exp(dt[..., None] * a) * h + (dt * x[:, t])[..., None] * bt
        y = (new * ct).sum(-1)
        if d is not None:
            y = y + d * x[:, t]
        if z is not None:
            y = y * F.silu(z[:, t])
        if live is not None:
            on = live > t
            new = torch.where(on[:, None, None], new, h)
            y = torch.where(on[:, None], y, torch.zeros_like(y))
        h = new
        rows.append(y)
    return (torch.stack(rows, 1) if rows else x.new_zeros(batch, 0, channels)), h


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """(y, x + residual)."""
    s = x if residual is None else x + residual
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight), s


def int4_weight(packed, scales, zeros=None):
    """The weight (outputs, inputs) that codes, scales and zero points stand for."""
    codes = torch.empty(packed.shape[0], 2 * packed.shape[1], dtype=torch.float64)
    codes[:, 0::2] = (packed & 15).double()
    codes[:, 1::2] = (packed >> 4).double()
    each = codes.shape[1] // scales.shape[1]
    zero = 8.0 if zeros is None else zeros.double().repeat_interleave(each, 1)
    return (codes - zero) * scales.double().repeat_interleave(each, 1)
