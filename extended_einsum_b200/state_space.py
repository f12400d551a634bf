"""A stack of selective state space layers on the sequence operators: training, prompts and single tokens.

One layer:

    s      = residual + x                          (ops.rms_norm, which also gives norm(s))
    v, z   = split(norm(s) W_in)
    v      = silu(causal convolution of v)         (ops.causal_conv1d)
    d, b, c = split(v W_x)
    v      = scan(v, d W_dt, b, c) * silu(z)       (ops.selective_scan)
    x      = v W_out

``SelectiveStack.forward`` trains (every operator has a backward pass; the projections are matrix products
of torch).  ``quantize`` gives a ``QuantizedStack``: the projections' weights in 4 bits, the norms'
outputs in 8, and a state per sequence that ``prompt`` fills and ``step`` carries on token by token.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import ops


@dataclass(frozen=True)
class StackShape:
    layers: int
    width: int  # of the residual stream
    channels: int  # of the convolution and the scan
    states: int = 16
    taps: int = 4
    rank: int = 32  # of the step sizes' projection, a multiple of 32
    outputs: int = 256  # logits per token


def init_parameters(shape: StackShape, generator: torch.Generator, device: str | torch.device = "cuda") -> dict:
    """Random parameters: decays 1 .. states, step sizes between 0.001 and 0.1."""

    def normal(*size, scale):
        return (scale * torch.randn(*size, generator=generator)).to(device)

    layers = []
    for _ in range(shape.layers):
        step = torch.exp(torch.rand(shape.channels, generator=generator) * math.log(100.0) + math.log(0.001))
        layers.append({
            "norm": torch.ones(shape.width, device=device),
            "w_in": normal(2 * shape.channels, shape.width, scale=shape.width**-0.5),
            "taps": normal(shape.channels, shape.taps, scale=shape.taps**-0.5),
            "taps_bias": torch.zeros(shape.channels, device=device),
            "w_x": normal(shape.rank + 2 * shape.states, shape.channels, scale=shape.channels**-0.5),
            "w_dt": normal(shape.channels, shape.rank, scale=shape.rank**-0.5),
            "dt_bias": torch.log(torch.expm1(step)).to(device),
            "log_a": torch.log(torch.arange(1, shape.states + 1).float()).repeat(shape.channels, 1).to(device),
            "d": torch.ones(shape.channels, device=device),
            "w_out": normal(shape.width, shape.channels, scale=shape.channels**-0.5),
        })
    return {
        "embedding": normal(shape.outputs, shape.width, scale=1.0),
        "layers": layers,
        "norm": torch.ones(shape.width, device=device),
        "w_logits": normal(shape.outputs, shape.width, scale=shape.width**-0.5),
    }


class SelectiveStack:
    """Training and whole sequences; activations of ``dtype``, the residual stream and the parameters float32."""

    def __init__(self, shape: StackShape, parameters: dict, dtype: torch.dtype = torch.bfloat16) -> None:
        self.shape, self.parameters, self.dtype = shape, parameters, dtype

    def tensors(self) -> list[torch.Tensor]:
        p = self.parameters
        return [p["embedding"], *(t for layer in p["layers"] for t in layer.values()), p["norm"], p["w_logits"]]

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        """Logits (batch, length, outputs) of whole numbers (batch, length)."""
        p, shape, dtype = self.parameters, self.shape, self.dtype
        residual = p["embedding"][tokens]
        x = torch.zeros_like(residual, dtype=dtype)
        for w in p["layers"]:
            y, residual = ops.rms_norm(x, w["norm"], residual=residual)
            v, z = (y @ w["w_in"].to(dtype).t()).split(shape.channels, dim=2)
            v = ops.causal_conv1d(v, w["taps"], w["taps_bias"], activation="silu")
            low, b, c = (v @ w["w_x"].to(dtype).t()).split([shape.rank, shape.states, shape.states], dim=2)
            v = ops.selective_scan(v, low @ w["w_dt"].to(dtype).t(), -torch.exp(w["log_a"]), b, c, w["d"], z=z,
                                   delta_bias=w["dt_bias"], softplus=True)
            x = v @ w["w_out"].to(dtype).t()
        y, _ = ops.rms_norm(x, p["norm"], residual=residual)
        return y @ p["w_logits"].to(dtype).t()

    def quantize(self, group: int = 32) -> QuantizedStack:
        return QuantizedStack(self, group)


class QuantizedStack:
    """Prompts and single tokens with 4-bit projections (``group`` inputs to a scale)."""

    def __init__(self, stack: SelectiveStack, group: int) -> None:
        self.shape, self.dtype = stack.shape, stack.dtype
        self.embedding, self.norm = stack.parameters["embedding"].detach(), stack.parameters["norm"].detach()

        def pack(w):
            return ops.int4_quantize(w.detach(), group, scale_dtype=torch.float32)

        self.logits = pack(stack.parameters["w_logits"])
        self.layers = []
        for w in stack.parameters["layers"]:
            kept = {k: t.detach() for k, t in w.items() if not k.startswith("w_")}
            kept["a"] = -torch.exp(kept.pop("log_a"))
            self.layers.append({**kept, **{k: pack(w[k]) for k in ("w_in", "w_x", "w_dt", "w_out")}})

    def empty_state(self, batch: int) -> list[dict]:
        """What a sequence carries between tokens, for each layer; zero before the first one."""
        s, device = self.shape, self.embedding.device
        return [
            {
                "taps": torch.zeros(batch, s.taps - 1, s.channels, device=device, dtype=self.dtype),
                "scan": torch.zeros(batch, s.channels, s.states, device=device),
            }
            for _ in range(s.layers)
        ]

    def _project(self, x, weight, x_scale=None):
        return ops.int4_linear(x, *weight, x_scale=x_scale, dtype=self.dtype)

    def _run(self, tokens, state, lengths):
        """One pass over (batch, length) tokens, or over (batch,) single ones (``lengths`` None)."""
        s, single = self.shape, tokens.dim() == 1
        residual = self.embedding[tokens]
        x = torch.zeros_like(residual, dtype=self.dtype)
        for w, held in zip(self.layers, state):
            q, scale, residual = ops.rms_norm(x, w["norm"], residual=residual, quantize="e4m3")
            v, z = self._project(q, w["w_in"], scale).split(s.channels, dim=-1)
            if single:
                v = ops.causal_conv1d_step(held["taps"], v, w["taps"], w["taps_bias"], activation="silu")
            else:
                v, held["taps"] = ops.causal_conv1d(v, w["taps"], w["taps_bias"], activation="silu", state=held["taps"],
                                                    lengths=lengths, return_state=True)
            low, b, c = self._project(v, w["w_x"]).split([s.rank, s.states, s.states], dim=-1)
            delta = self._project(low, w["w_dt"])
            if single:
                v = ops.selective_scan_step(held["scan"], v, delta, w["a"], b, c, w["d"], z=z, delta_bias=w["dt_bias"],
                                            softplus=True)
            else:
                v, held["scan"] = ops.selective_scan(v, delta, w["a"], b, c, w["d"], z=z, delta_bias=w["dt_bias"], softplus=True,
                                                     state=held["scan"], lengths=lengths, return_state=True)
            x = self._project(v, w["w_out"])
        q, scale, _ = ops.rms_norm(x, self.norm, residual=residual, quantize="e4m3")
        return self._project(q, self.logits, scale)

    @torch.no_grad()
    def prompt(self, tokens: torch.Tensor, state: list[dict], lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Logits (batch, length, outputs); ``state`` moves past the tokens (past each sequence's first
        ``lengths`` ones)."""
        return self._run(tokens, state, lengths)

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, state: list[dict]) -> torch.Tensor:
        """Logits (batch, outputs) after one more token (batch,) of every sequence."""
        return self._run(tokens, state, None)
