"""Workloads of the sequence operators: the selective state space scan with its short causal
convolution, the root-mean-square norm with the residual's addition and 8-bit outputs, and the
products with 4-bit weights.

Each case is one call of one operator.  ``run`` computes it in a plain form (elementary torch
operations in float32, rounded once at the end) or, with ``own`` set, through
``extended_einsum_b200.ops`` as a user's program does.  Layouts are channel-last: (batch, length,
channels).

The recurrence, for every channel d and state n:

    delta = softplus(raw + bias_d)
    h_t   = exp(delta_t A_dn) h_{t-1} + delta_t B_tn x_td
    y_t   = (sum_n C_tn h_t + D_d x_td) * silu(z_td)

the convolution in front of it y_t = silu(bias + sum_j w_j x_{t-W+1+j}), the norm
y = (x + residual) * rsqrt(mean((x + residual)^2) + eps) * w, and the 4-bit product
y_mo = sum_k x_mk s_og (q_ok - zero_og), g the group of k.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
E4M3_MAX = 448.0
INT8_MAX = 127.0
TINY = 2.0**-126


def listed():
    return [
        # the first tokens of three short prompts of unequal length, odd sizes, float32
        {"name": "scan_ragged_f32", "op": "scan", "dtype": "f32", "batch": 3, "length": 509, "channels": 1000,
         "states": 12, "groups": 1, "ragged": True},
        # four long prompts read at once: the largest case
        {"name": "scan_prompt_bf16", "op": "scan", "dtype": "bf16", "batch": 4, "length": 4096, "channels": 4096,
         "states": 16, "groups": 1, "ragged": False},
        # a training step's recurrence, forward and backward
        {"name": "scan_train_bf16", "op": "scan_train", "dtype": "bf16", "batch": 2, "length": 2048, "channels": 2048,
         "states": 16, "groups": 1},
        # one new token for each of 64 answers under way
        {"name": "scan_step_bf16", "op": "scan_step", "dtype": "bf16", "batch": 64, "channels": 4096, "states": 16,
         "groups": 1},
        # the convolution over the same four prompts
        {"name": "conv_prompt_bf16", "op": "conv", "dtype": "bf16", "batch": 4, "length": 4096, "channels": 4096,
         "width": 4, "ragged": False},
        # the convolution in training, odd sizes, float32
        {"name": "conv_train_f32", "op": "conv_train", "dtype": "f32", "batch": 3, "length": 1021, "channels": 1000,
         "width": 3},
        # the norm before the projection of a single token, quantised for it: where latency counts
        {"name": "norm_token_e4m3", "op": "norm", "dtype": "bf16", "rows": 1, "columns": 4096, "quantize": "e4m3"},
        # the same over prompts
        {"name": "norm_prompt_e4m3", "op": "norm", "dtype": "bf16", "rows": 16384, "columns": 4096,
         "quantize": "e4m3"},
        # the norm in training, an odd number of rows and a width that fills no power of two
        {"name": "norm_train_bf16", "op": "norm_train", "dtype": "bf16", "rows": 4099, "columns": 2560},
        # a projection of a single token
        {"name": "int4_token_bf16", "op": "int4", "dtype": "bf16", "rows": 1, "inputs": 4096, "outputs": 8192,
         "group": 128, "zeros": False, "quantize": "none"},
        # a larger one for 16 answers under way, activations in 8 bits, zero points
        {"name": "int4_rows16_e4m3", "op": "int4", "dtype": "bf16", "rows": 16, "inputs": 8192, "outputs": 16384,
         "group": 64, "zeros": True, "quantize": "e4m3"},
        # float32 activations, a few tokens, odd numbers of rows and outputs
        {"name": "int4_rows5_f32", "op": "int4", "dtype": "f32", "rows": 5, "inputs": 1056, "outputs": 2051,
         "group": 32, "zeros": True, "quantize": "none"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_train", "scan_step", "conv", "conv_train", "norm", "norm_train", "int4", "int4"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = {"op": op, "dtype": dtype}
    if op in ("scan", "scan_train"):
        case["states"] = rng.choice([16, 16, 16, 1, 4, 12, 24, 64])
        most = (1 << 28 if op == "scan" else 1 << 26) // (16 * max(1, -(-case["states"] // 16)))
        case["length"] = _spread(rng, 1, 16384)
        case["batch"] = _spread(rng, 1, max(1, min(16, most // case["length"])))
        case["groups"] = rng.choice([1, 1, 2])
        case["channels"] = case["groups"] * _spread(rng, 16, max(17, min(4096, most // (case["length"] * case["batch"])) // 2))
        if op == "scan":
            case["ragged"] = rng.random() < 0.4
    elif op == "scan_step":
        case["states"] = rng.choice([16, 16, 16, 1, 12, 64])
        case["batch"] = _spread(rng, 1, 256)
        case["groups"] = rng.choice([1, 1, 2])
        case["channels"] = case["groups"] * _spread(rng, 32, 4096)
    elif op in ("conv", "conv_train"):
        case["length"] = _spread(rng, 1, 16384)
        case["batch"] = _spread(rng, 1, 16)
        case["channels"] = _spread(rng, 16, max(17, min(8192, (1 << 26) // (case["length"] * case["batch"]))))
        case["width"] = rng.choice([4, 4, 3, 2])
        if op == "conv":
            case["ragged"] = rng.random() < 0.4
    elif op in ("norm", "norm_train"):
        case["columns"] = _spread(rng, 32, 16384)
        case["rows"] = _spread(rng, 1, max(2, (1 << 26) // case["columns"]))
        if op == "norm":
            case["quantize"] = rng.choice(["none", "e4m3", "e4m3", "int8"])
    else:
        case["group"] = rng.choice([32, 64, 128, 128])
        case["inputs"] = case["group"] * _spread(rng, 2, 16384 // case["group"])
        case["outputs"] = _spread(rng, 16, 16384)
        case["rows"] = _spread(rng, 1, 64)
        case["zeros"] = rng.random() < 0.5
        case["quantize"] = rng.choice(["none", "none", "e4m3"])
    return case


# ---------------------------------------------------------------------------
# inputs


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _lengths(gen, case):
    """None, or unequal lengths: one whole, the others anywhere from nothing to whole."""
    if not case.get("ragged"):
        return None
    lengths = torch.randint(0, case["length"] + 1, (case["batch"],), generator=gen, device="cuda", dtype=torch.int32)
    lengths[0] = case["length"]
    return lengths


def _scan_parameters(gen, channels, states):
    """A as a decay spectrum 1..states with some spread, D near one, and a bias whose softplus lies in 0.001 .. 0.1."""
    spectrum = torch.arange(1, states + 1, device="cuda", dtype=torch.float32)
    a = -spectrum * torch.exp(0.2 * torch.randn(channels, states, generator=gen, device="cuda"))
    d = 1.0 + 0.1 * torch.randn(channels, generator=gen, device="cuda")
    step = torch.exp(torch.rand(channels, generator=gen, device="cuda") * math.log(100.0) + math.log(0.001))
    return a, d, torch.log(torch.expm1(step))


def _int4_codes(state):
    packed = state["packed"].to(torch.int32)
    return torch.stack([packed & 15, packed >> 4], dim=2).reshape(packed.shape[0], -1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if op in ("scan", "scan_train"):
        b, t, c, n, g = (case[k] for k in ("batch", "length", "channels", "states", "groups"))
        # x is the convolution's output; z the other half of a projection's output, so a strided view
        s["x"] = _randn(gen, b, t, c, dtype=dtype)
        s["z"] = _randn(gen, b, t, 2 * c, dtype=dtype)[:, :, c:]
        s["delta"] = _randn(gen, b, t, c, dtype=dtype, scale=0.5)
        both = _randn(gen, b, t, 2, g, n, dtype=dtype)
        s["b"], s["c"] = both[:, :, 0], both[:, :, 1]
        s["a"], s["d"], s["delta_bias"] = _scan_parameters(gen, c, n)
        if op == "scan":
            s["lengths"] = _lengths(gen, case)
            s["state"] = _randn(gen, b, c, n)
        else:
            s["dy"] = _randn(gen, b, t, c, dtype=dtype)
    elif op == "scan_step":
        b, c, n, g = (case[k] for k in ("batch", "channels", "states", "groups"))
        s["x"] = _randn(gen, b, c, dtype=dtype)
        s["z"] = _randn(gen, b, 2 * c, dtype=dtype)[:, c:]
        s["delta"] = _randn(gen, b, c, dtype=dtype, scale=0.5)
        both = _randn(gen, b, 2, g, n, dtype=dtype)
        s["b"], s["c"] = both[:, 0], both[:, 1]
        s["a"], s["d"], s["delta_bias"] = _scan_parameters(gen, c, n)
        s["state"] = _randn(gen, b, c, n)
    elif op in ("conv", "conv_train"):
        b, t, c, w = (case[k] for k in ("batch", "length", "channels", "width"))
        s["x"] = _randn(gen, b, t, 2 * c, dtype=dtype)[:, :, :c]  # the first half of a projection's output
        s["weight"] = _randn(gen, c, w, scale=1.0 / math.sqrt(w))
        s["bias"] = _randn(gen, c, scale=0.1)
        if op == "conv":
            s["lengths"] = _lengths(gen, case)
            s["state"] = _randn(gen, b, w - 1, c, dtype=dtype)
        else:
            s["dy"] = _randn(gen, b, t, c, dtype=dtype)
    elif op in ("norm", "norm_train"):
        r, c = case["rows"], case["columns"]
        s["x"] = _randn(gen, r, c, dtype=dtype)
        s["residual"] = _randn(gen, r, c, dtype=dtype, scale=2.0)
        s["weight"] = 1.0 + _randn(gen, c, scale=0.1)
        if op == "norm_train":
            s["dy"] = _randn(gen, r, c, dtype=dtype)
            s["dsum"] = _randn(gen, r, c, dtype=dtype)
    else:
        r, k, o, group = case["rows"], case["inputs"], case["outputs"], case["group"]
        s["packed"] = torch.randint(0, 256, (o, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(o, k // group, generator=gen, device="cuda")) / (8.0 * math.sqrt(k))).to(
            dtype if dtype != torch.float32 else torch.float32)
        s["zeros"] = None
        if case["zeros"]:
            s["zeros"] = torch.randint(4, 12, (o, k // group), generator=gen, device="cuda", dtype=torch.uint8)
        x = _randn(gen, r, k)
        s["x_scale"] = None
        if case["quantize"] == "e4m3":
            s["x_scale"] = x.abs().amax(1) / E4M3_MAX
            s["x"] = (x / s["x_scale"][:, None]).to(torch.float8_e4m3fn)
        else:
            s["x"] = x.to(dtype)
    return s


# ---------------------------------------------------------------------------
# the plain forms


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(torch.minimum(v, torch.full_like(v, 20.0)))))


def _recurrence(decay, drive):
    """h_t = decay_t h_{t-1} + drive_t along axis 1, by doubling: log2(length) steps over the whole length."""
    length, k = decay.shape[1], 1
    while k < length:
        drive = torch.cat([drive[:, :k], drive[:, k:] + decay[:, k:] * drive[:, :-k]], dim=1)
        decay = torch.cat([decay[:, :k], decay[:, k:] * decay[:, :-k]], dim=1)
        k *= 2
    return drive


def _per_channel(v, channels):
    """(batch, length, groups, states) seen by each channel."""
    return v.repeat_interleave(channels // v.shape[2], dim=2)


def _masked(s):
    """Truth values (batch, length, 1): the positions that are part of their sequence."""
    x = s["x"]
    at = torch.arange(x.shape[1], device=x.device)
    return (at[None, :] < s["lengths"][:, None])[:, :, None]


def _plain_scan(s):
    dtype, channels = s["x"].dtype, s["x"].shape[2]
    x, z = s["x"].float(), s["z"].float()
    delta = _softplus(s["delta"].float() + s["delta_bias"])
    if s["lengths"] is not None:
        delta = torch.where(_masked(s), delta, torch.zeros_like(delta))
    decay = torch.exp(delta[..., None] * s["a"])
    drive = (delta * x)[..., None] * _per_channel(s["b"].float(), channels)
    drive[:, 0] += decay[:, 0] * s["state"]
    h = _recurrence(decay, drive)
    last = h[:, -1].clone()
    y = (h * _per_channel(s["c"].float(), channels)).sum(-1) + s["d"] * x
    y = y * _silu(z)
    if s["lengths"] is not None:
        y = torch.where(_masked(s), y, torch.zeros_like(y))
    return {"y": y.to(dtype), "state": last}


def _plain_scan_train(s):
    dtype, channels = s["x"].dtype, s["x"].shape[2]
    x, z, dy = s["x"].float(), s["z"].float(), s["dy"].float()
    raw = s["delta"].float() + s["delta_bias"]
    delta = _softplus(raw)
    b, c = _per_channel(s["b"].float(), channels), _per_channel(s["c"].float(), channels)
    decay = torch.exp(delta[..., None] * s["a"])
    h = _recurrence(decay, (delta * x)[..., None] * b)
    y = (h * c).sum(-1) + s["d"] * x
    sig = 1.0 / (1.0 + torch.exp(-z))
    out = y * z * sig
    dz = dy * y * sig * (1.0 + z * (1.0 - sig))
    dv = dy * z * sig
    # the adjoint runs the same recurrence backwards: g_t = C_t dv_t + decay_{t+1} g_{t+1}
    later = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], dim=1)
    g = _recurrence(later.flip(1), (dv[..., None] * c).flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], dim=1)
    through = g * before * decay
    into = (g * b).sum(-1)
    ddelta = (through * s["a"]).sum(-1) + into * x
    draw_ = ddelta / (1.0 + torch.exp(-raw))
    shape = (*s["b"].shape[:3], channels // s["b"].shape[2], s["b"].shape[3])
    db = (g * (delta * x)[..., None]).reshape(shape).sum(3)
    dc = (h * dv[..., None]).reshape(shape).sum(3)
    return {
        "y": out.to(dtype),
        "dx": (dv * s["d"] + into * delta).to(dtype),
        "ddelta": draw_.to(dtype),
        "da": (through * delta[..., None]).sum((0, 1)),
        "db": db.to(dtype),
        "dc": dc.to(dtype),
        "dd": (dv * x).sum((0, 1)),
        "dz": dz.to(dtype),
        "ddelta_bias": draw_.sum((0, 1)),
    }


def _plain_scan_step(s):
    x, z = s["x"].float(), s["z"].float()
    channels = x.shape[1]
    delta = _softplus(s["delta"].float() + s["delta_bias"])
    b = _per_channel(s["b"].float()[:, None], channels)[:, 0]
    c = _per_channel(s["c"].float()[:, None], channels)[:, 0]
    s["state"].copy_(torch.exp(delta[..., None] * s["a"]) * s["state"] + (delta * x)[..., None] * b)
    y = ((s["state"] * c).sum(-1) + s["d"] * x) * _silu(z)
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _windows(s, before):
    """The convolution's sums before the activation, and the sequence with the `width - 1` values before it."""
    length, width = s["x"].shape[1], s["weight"].shape[1]
    full = torch.cat([before, s["x"].float()], dim=1)
    taps = torch.arange(length, device=full.device)[:, None] + torch.arange(width, device=full.device)
    return (full[:, taps] * s["weight"].t()).sum(2) + s["bias"], full


def _plain_conv(s):
    dtype, width = s["x"].dtype, s["weight"].shape[1]
    pre, full = _windows(s, s["state"].float())
    y = _silu(pre)
    if s["lengths"] is None:
        return {"y": y.to(dtype), "state": full[:, full.shape[1] - (width - 1):].to(dtype)}
    y = torch.where(_masked(s), y, torch.zeros_like(y))
    rows = s["lengths"].long()[:, None] + torch.arange(width - 1, device=y.device)
    last = full.gather(1, rows[:, :, None].expand(-1, -1, full.shape[2]))
    return {"y": y.to(dtype), "state": last.to(dtype)}


def _plain_conv_train(s):
    dtype, width, length = s["x"].dtype, s["weight"].shape[1], s["x"].shape[1]
    zero = torch.zeros(s["x"].shape[0], width - 1, s["x"].shape[2], device=s["x"].device)
    pre, full = _windows(s, zero)
    sig = 1.0 / (1.0 + torch.exp(-pre))
    dpre = s["dy"].float() * sig * (1.0 + pre * (1.0 - sig))
    taps = torch.arange(length, device=full.device)[:, None] + torch.arange(width, device=full.device)
    dweight = (full[:, taps] * dpre[:, :, None]).sum((0, 1)).t()
    after = torch.cat([dpre, zero], dim=1)
    dx = (after[:, taps] * s["weight"].flip(1).t()).sum(2)
    return {"y": (pre * sig).to(dtype), "dx": dx.to(dtype), "dweight": dweight, "dbias": dpre.sum((0, 1))}


def _plain_norm(s):
    dtype, quantize = s["x"].dtype, s["case"]["quantize"]
    total = s["x"].float() + s["residual"].float()
    y = total * torch.rsqrt((total * total).mean(1, keepdim=True) + EPS) * s["weight"]
    if quantize == "none":
        return {"y": y.to(dtype), "sum": total.to(dtype)}
    most = E4M3_MAX if quantize == "e4m3" else INT8_MAX
    scale = torch.clamp(y.abs().amax(1) / most, min=TINY)
    codes = y / scale[:, None]
    if quantize == "e4m3":
        return {"q": codes.to(torch.float8_e4m3fn), "scale": scale, "sum": total.to(dtype)}
    return {"q": _worth(torch.round(codes).to(torch.int8), scale), "scale": scale, "sum": total.to(dtype)}


def _worth(codes, scale):
    """The values that whole 8-bit codes stand for."""
    return (codes.float() * scale[:, None]).to(torch.bfloat16)


def _plain_norm_train(s):
    dtype = s["x"].dtype
    total = s["x"].float() + s["residual"].float()
    r = torch.rsqrt((total * total).mean(1, keepdim=True) + EPS)
    unit = total * r
    dy = s["dy"].float()
    du = dy * s["weight"]
    dtotal = r * (du - unit * (du * unit).mean(1, keepdim=True)) + s["dsum"].float()
    return {"y": (unit * s["weight"]).to(dtype), "sum": total.to(dtype), "dx": dtotal.to(dtype),
            "dresidual": dtotal.to(dtype), "dweight": (dy * unit).sum(0)}


def _plain_int4(s):
    codes = _int4_codes(s)
    group = s["case"]["group"]
    zero = s["zeros"].float() if s["zeros"] is not None else torch.full_like(s["scales"], 8.0, dtype=torch.float32)
    w = codes.float().reshape(codes.shape[0], -1, group) - zero[:, :, None]
    w = (w * s["scales"].float()[:, :, None]).reshape(codes.shape)
    y = s["x"].float() @ w.t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None]
    return {"y": y.to(DTYPES[s["case"]["dtype"]])}


PLAIN = {"scan": _plain_scan, "scan_train": _plain_scan_train, "scan_step": _plain_scan_step, "conv": _plain_conv,
         "conv_train": _plain_conv_train, "norm": _plain_norm, "norm_train": _plain_norm_train, "int4": _plain_int4}


# ---------------------------------------------------------------------------
# the framework's operators


def _own_scan(ops, s):
    y, state = ops.selective_scan(
        s["x"], s["delta"], s["a"], s["b"], s["c"], s["d"], z=s["z"], delta_bias=s["delta_bias"], softplus=True,
        state=s["state"], lengths=s["lengths"], return_state=True)
    return {"y": y, "state": state}


def _own_scan_train(ops, s):
    names = ("x", "delta", "a", "b", "c", "d", "z", "delta_bias")
    v = {k: s[k].detach().requires_grad_() for k in names}
    y = ops.selective_scan(v["x"], v["delta"], v["a"], v["b"], v["c"], v["d"], z=v["z"], delta_bias=v["delta_bias"],
                           softplus=True)
    grads = torch.autograd.grad(y, [v[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def _own_scan_step(ops, s):
    y = ops.selective_scan_step(s["state"], s["x"], s["delta"], s["a"], s["b"], s["c"], s["d"], z=s["z"],
                                delta_bias=s["delta_bias"], softplus=True)
    return {"y": y, "state": s["state"]}


def _own_conv(ops, s):
    y, state = ops.causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu", state=s["state"],
                                 lengths=s["lengths"], return_state=True)
    return {"y": y, "state": state}


def _own_conv_train(ops, s):
    x, weight, bias = (s[k].detach().requires_grad_() for k in ("x", "weight", "bias"))
    y = ops.causal_conv1d(x, weight, bias, activation="silu")
    dx, dweight, dbias = torch.autograd.grad(y, [x, weight, bias], s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}


def _own_norm(ops, s):
    quantize = s["case"]["quantize"]
    if quantize == "none":
        y, total = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return {"y": y, "sum": total}
    q, scale, total = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, quantize=quantize)
    return {"q": q if quantize == "e4m3" else _worth(q, scale), "scale": scale, "sum": total}


def _own_norm_train(ops, s):
    x, residual, weight = (s[k].detach().requires_grad_() for k in ("x", "residual", "weight"))
    y, total = ops.rms_norm(x, weight, residual=residual, eps=EPS)
    dx, dresidual, dweight = torch.autograd.grad([y, total], [x, residual, weight], [s["dy"], s["dsum"]])
    return {"y": y.detach(), "sum": total.detach(), "dx": dx, "dresidual": dresidual, "dweight": dweight}


def _own_int4(ops, s):
    y = ops.int4_linear(s["x"], s["packed"], s["scales"], s["zeros"], x_scale=s["x_scale"],
                        dtype=DTYPES[s["case"]["dtype"]])
    return {"y": y}


OWN = {"scan": _own_scan, "scan_train": _own_scan_train, "scan_step": _own_scan_step, "conv": _own_conv,
       "conv_train": _own_conv_train, "norm": _own_norm, "norm_train": _own_norm_train, "int4": _own_int4}


def run(state):
    op = state["case"]["op"]
    if own:
        from extended_einsum_b200 import ops

        return OWN[op](ops, state)
    return PLAIN[op](state)


# ---------------------------------------------------------------------------
# what one pass has to move and compute


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op in ("scan", "scan_train"):
        b, t, c, n, g = (case[k] for k in ("batch", "length", "channels", "states", "groups"))
        tokens = b * t
        if case.get("ragged"):  # the lengths are uniform, one of them whole
            tokens = t * (1 + (b - 1) / 2)
        rows = tokens * c * size
        shared = tokens * 2 * g * n * size
        parameters = (c * n + 2 * c) * 4
        if op == "scan":  # x, delta, z in; y out; B and C; the state in and out.  6 operations per state, 10 per channel
            return {"bytes": 4 * rows + shared + parameters + 2 * b * c * n * 4, "flops": tokens * c * (6 * n + 10)}
        # both directions: x, delta, z and dy in, y, dx, ddelta and dz out; B, C and their gradients
        return {"bytes": 8 * rows + 2 * shared + 2 * parameters, "flops": tokens * c * (24 * n + 40)}
    if op == "scan_step":
        b, c, n, g = (case[k] for k in ("batch", "channels", "states", "groups"))
        return {"bytes": 4 * b * c * size + 2 * b * g * n * size + (c * n + 2 * c) * 4 + 2 * b * c * n * 4,
                "flops": b * c * (6 * n + 10)}
    if op in ("conv", "conv_train"):
        b, t, c, w = (case[k] for k in ("batch", "length", "channels", "width"))
        tokens = b * t if not case.get("ragged") else t * (1 + (b - 1) / 2)
        rows = tokens * c * size
        parameters = c * (w + 1) * 4
        if op == "conv":
            return {"bytes": 2 * rows + parameters + 2 * b * (w - 1) * c * size, "flops": tokens * c * (2 * w + 5)}
        return {"bytes": 4 * rows + 2 * parameters, "flops": tokens * c * (8 * w + 15)}
    if op == "norm":
        r, c = case["rows"], case["columns"]
        out = size if case["quantize"] == "none" else 1
        return {"bytes": r * c * (3 * size + out) + (0 if case["quantize"] == "none" else 4 * r) + 4 * c,
                "flops": r * c * 6}
    if op == "norm_train":  # x, residual, dy and dsum in, y, the sum and the gradient that x and residual share out
        r, c = case["rows"], case["columns"]
        return {"bytes": r * c * 7 * size + 2 * 4 * c, "flops": r * c * 16}
    r, k, o = case["rows"], case["inputs"], case["outputs"]
    groups = o * (k // case["group"])
    x = r * k * (size if case["quantize"] == "none" else 1) + (0 if case["quantize"] == "none" else 4 * r)
    return {"bytes": o * k / 2 + groups * size + (groups if case["zeros"] else 0) + x + r * o * size,
            "flops": 2 * r * k * o}


# ---------------------------------------------------------------------------
# the definitions in 64 bits: the recurrence token by token, gradients by differentiating it


def _exact_scan(s, wanted):
    """Outputs, last state and (if wanted) gradients of the recurrence taken one token at a time."""
    names = ("x", "delta", "a", "b", "c", "d", "z", "delta_bias")
    v = {k: s[k].double().requires_grad_(wanted) for k in names}
    batch, length, channels = v["x"].shape
    each = channels // v["b"].shape[2]
    h = s["state"].double() if s.get("state") is not None else torch.zeros(
        batch, channels, v["a"].shape[1], device="cuda", dtype=torch.float64)
    rows = []
    for t in range(length):
        xt, zt = v["x"][:, t], v["z"][:, t]
        step = torch.nn.functional.softplus(v["delta"][:, t] + v["delta_bias"], threshold=40.0)
        b, c = (v[k][:, t].repeat_interleave(each, dim=1) for k in ("b", "c"))
        new = torch.exp(step.unsqueeze(2) * v["a"]) * h + (step * xt).unsqueeze(2) * b
        y = (torch.einsum("bcn,bcn->bc", new, c) + v["d"] * xt) * torch.nn.functional.silu(zt)
        if s.get("lengths") is not None:
            live = (s["lengths"] > t)
            new, y = torch.where(live[:, None, None], new, h), torch.where(live[:, None], y, 0.0)
        h = new
        rows.append(y)
    y = torch.stack(rows, dim=1)
    if not wanted:
        return {"y": y, "state": h}
    grads = torch.autograd.grad(y, [v[k] for k in names], s["dy"].double())
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def _exact_conv(s, wanted):
    x, weight, bias = (s[k].double().requires_grad_(wanted) for k in ("x", "weight", "bias"))
    batch, length, channels = x.shape
    width = weight.shape[1]
    before = s["state"].double() if s.get("state") is not None else x.new_zeros(batch, width - 1, channels)
    full = torch.cat([before, x], dim=1)
    y = bias.expand(batch, length, channels)
    for j in range(width):
        y = y + weight[:, j] * full[:, j : j + length]
    y = torch.nn.functional.silu(y)
    if wanted:
        dx, dweight, dbias = torch.autograd.grad(y, [x, weight, bias], s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}
    ends = [length] * batch if s["lengths"] is None else s["lengths"].tolist()
    for i, end in enumerate(ends):
        y[i, end:] = 0.0
    return {"y": y, "state": torch.stack([full[i, end : end + width - 1] for i, end in enumerate(ends)])}


def _exact_norm(s, wanted):
    x, residual, weight = (s[k].double().requires_grad_(wanted) for k in ("x", "residual", "weight"))
    total = x + residual
    y = weight * total / torch.sqrt(torch.linalg.vector_norm(total, dim=1, keepdim=True) ** 2 / total.shape[1] + EPS)
    if wanted:
        dx, dresidual, dweight = torch.autograd.grad([y, total], [x, residual, weight], [s["dy"].double(), s["dsum"].double()])
        return {"y": y.detach(), "sum": total.detach(), "dx": dx, "dresidual": dresidual, "dweight": dweight}
    quantize = s["case"]["quantize"]
    if quantize == "none":
        return {"y": y, "sum": total}
    scale = torch.linalg.vector_norm(y, ord=float("inf"), dim=1) / (E4M3_MAX if quantize == "e4m3" else INT8_MAX)
    return {"q": y / scale[:, None] if quantize == "e4m3" else y, "scale": scale, "sum": total}


def _exact_int4(s):
    packed = s["packed"].cpu().numpy()
    codes = torch.empty(packed.shape[0], 2 * packed.shape[1], device="cuda", dtype=torch.float64)
    codes[:, 0::2] = torch.from_numpy(packed % 16).cuda().double()
    codes[:, 1::2] = torch.from_numpy(packed // 16).cuda().double()
    each = codes.shape[1] // s["scales"].shape[1]
    codes -= 8.0 if s["zeros"] is None else s["zeros"].double().repeat_interleave(each, dim=1)
    codes *= s["scales"].double().repeat_interleave(each, dim=1)
    x = s["x"].double() if s["x_scale"] is None else s["x"].float().double() * s["x_scale"].double()[:, None]
    return {"y": torch.einsum("mk,ok->mo", x, codes)}


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op in ("scan", "scan_train"):
        # the differentiated recurrence keeps a few 64-bit states per token
        if op == "scan_train" and case["batch"] * case["length"] * case["channels"] * case["states"] > 1 << 28:
            return None
        return _exact_scan(s, op == "scan_train")
    if op == "scan_step":
        one = {**s, **{k: s[k][:, None] for k in ("x", "z", "delta", "b", "c")}}
        out = _exact_scan(one, False)
        return {"y": out["y"][:, 0], "state": out["state"]}
    if op in ("conv", "conv_train"):
        return _exact_conv(s, op == "conv_train")
    if op in ("norm", "norm_train"):
        return _exact_norm(s, op == "norm_train")
    return _exact_int4(s)
