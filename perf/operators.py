"""A surfel decoder's operators, as measurable cases.

A decoder turns a latent vector per surfel into the appearance values that
the renderers take (18 classic or 57 neural values): layer norm, linear
layers and activations over as many rows as there are surfels, trained
through the renderer. Its activations are kept in 8 bits for the backward
pass. Each case is one pass through one operator:

* ``layer_norm``: the forward and backward pass (or the forward alone), the
  input kept in its own type or in 8 bits;
* ``checkpoint``: rows written to 8 bits and read back;
* ``activation``: the forward and backward pass, the input kept in 8 bits;
* ``linear``: the forward and backward pass, the input kept in 8 bits for the
  weight's gradient, or the forward alone.

Row counts are the surfel counts of ``workloads.py`` (1,024 to a million)
and those of a few surfels decoded at a time; widths are generic.

The 8-bit form of a group of 32 consecutive features of a row (the last group
of a row may be shorter) is q 2^e with e the smallest integer, at least
``LEAST_EXPONENT`` of the type, for which the group's largest magnitude
rounds to at most 127, and q the values over 2^e rounded to the nearest, ties
to even.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

GROUP = 32
EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
# float16's values are multiples of 2^-24, the others' exponents end at -126.
LEAST_EXPONENT = {torch.float32: -126, torch.bfloat16: -126, torch.float16: -24}
LIMIT_VALUES = 1_000_000 * 512   # rows * widest side of a drawn case
LIMIT_FLOPS = 6.0 * 1_000_000 * 512 * 512


def _case(name, op, rows, features, dtype="bfloat16", outputs=0, train=True, eight=True,
          kind="", weights=""):
    return dict(name=name, op=op, rows=rows, features=features, dtype=dtype, outputs=outputs,
                train=train, eight=eight, kind=kind, weights=weights or dtype)


def listed():
    return [
        # Layer norm of the smallest workload's latents, in the renderer's own
        # type, trained: launches and host time count.
        _case("norm_small", "layer_norm", 1_024, 64, "float32", eight=False),
        # A mid-sized scene's latents, in bfloat16 with float32 parameters.
        _case("norm_mid", "layer_norm", 100_000, 256, eight=False, weights="float32"),
        # A width that no vector load divides, 8-bit kept input.
        _case("norm_ragged", "layer_norm", 33_333, 187, "float16"),
        # The largest scene with wide latents, 8-bit kept input.
        _case("norm_large", "layer_norm", 1_000_000, 512),
        # Keeping latents of a mid-sized scene in 8 bits and reading them back.
        _case("checkpoint_mid", "checkpoint", 100_000, 256, "float32"),
        _case("checkpoint_large", "checkpoint", 1_000_000, 512),
        # The renderer's own sine activation on a few thousand surfels.
        _case("sine_small", "activation", 10_000, 128, "float32", kind="sine"),
        # A hidden layer of the largest scene.
        _case("gelu_large", "activation", 1_000_000, 512, kind="gelu"),
        # One surfel decoded (picking, editing): a single row, no gradients.
        _case("linear_row", "linear", 1, 1_024, outputs=1_024, train=False),
        # The head that gives the neural renderer's 57 values, in its type.
        _case("head_small", "linear", 1_024, 64, "float32", outputs=57),
        # A hidden layer of a mid-sized scene.
        _case("linear_mid", "linear", 100_000, 256, outputs=256),
        # A hidden layer of the largest scene.
        _case("linear_large", "linear", 1_000_000, 512, outputs=512),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def draw(rng):
    """Any operator, type and size between the listed ones, odd ones among
    them."""
    while True:
        op = rng.choice(("layer_norm", "layer_norm", "checkpoint", "activation", "linear",
                         "linear"))
        rows = _log(rng, 1, 1_000_000)
        features = rng.choice((_log(rng, 8, 1_024), 32 * _log(rng, 1, 32)))
        dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
        case = _case("", op, rows, features, dtype)
        if op == "layer_norm":
            case["eight"] = rng.random() < 0.5
            case["weights"] = rng.choice((dtype, "float32"))
            case["train"] = rng.random() < 0.8
        elif op == "activation":
            case["kind"] = rng.choice(("sine", "gelu", "silu"))
        elif op == "linear":
            case["outputs"] = rng.choice((18, 57, _log(rng, 8, 1_024), 32 * _log(rng, 1, 32)))
            case["train"] = rng.random() < 0.8
        del case["name"]
        if rows * max(features, case["outputs"]) <= LIMIT_VALUES and \
                work(case)["flops"] <= LIMIT_FLOPS:
            return case


def work(case):
    rows, features, outputs = case["rows"], case["features"], case["outputs"]
    size = BYTES[case["dtype"]]
    values = rows * features
    kept = rows * (features + -(-features // GROUP)) * 2  # written once, read once
    if case["op"] == "checkpoint":
        return {"bytes": 2 * values * size + kept, "flops": 4 * values}
    if case["op"] == "activation":
        return {"bytes": 4 * values * size + kept, "flops": 20 * values}
    if case["op"] == "layer_norm":
        parameters = 2 * features * BYTES[case["weights"]]
        if not case["train"]:
            return {"bytes": 2 * values * size + parameters, "flops": 8 * values}
        return {"bytes": 4 * values * size + 2 * parameters + (kept if case["eight"] else 0),
                "flops": 24 * values}
    parameters = (outputs * features + outputs) * size
    sides = rows * (features + outputs) * size
    if not case["train"]:
        return {"bytes": sides + parameters, "flops": 2 * values * outputs}
    return {"bytes": 2 * sides + 2 * parameters + kept, "flops": 6 * values * outputs}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    rows, features = case["rows"], case["features"]
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=device) * 2 - 1

    state = dict(case=case)
    if case["op"] == "layer_norm":
        # Latents: rows with an offset of their own, and a few features that
        # are several times larger than the rest.
        scale = 1 + 7 * (uniform(features) > 0.96).float()
        x = normal(rows, features).mul_(scale).add_(normal(rows, 1) * 0.5)
        weights = DTYPES[case["weights"]]
        state["weight"] = (1 + 0.1 * normal(features)).to(weights)
        state["bias"] = (0.1 * normal(features)).to(weights)
        grads = (rows, features)
    elif case["op"] == "linear":
        outputs = case["outputs"]
        x = normal(rows, features)
        state["weight"] = (uniform(outputs, features) / math.sqrt(features)).to(dtype)
        state["bias"] = (uniform(outputs) / math.sqrt(features)).to(dtype)
        grads = (rows, outputs)
    else:
        # A sine layer's input is a thirtieth of its phase.
        x = normal(rows, features) / (30 if case["kind"] == "sine" else 1)
        grads = (rows, features)
    state["x"] = x.to(dtype)
    del x
    if case["op"] != "checkpoint" and case["train"]:
        state["grad"] = (normal(*grads) * 0.05).to(dtype)
        for name in ("x", "weight", "bias"):
            if name in state:
                state[name].requires_grad_()
    return state


# --------------------------------------------------------------------------
# The operators in their plain form


def _power(exponent):
    """2^exponent as float32, for int32 exponents in [-126, 127]."""
    return ((exponent + 127) << 23).view(torch.float32)


def _eight(values, least):
    """float32 rows as their 8-bit form stands for them."""
    rows, features = values.shape
    short = -features % GROUP
    groups = torch.nn.functional.pad(values, (0, short)).view(rows, -1, GROUP)
    largest = groups.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(largest)  # largest = mantissa 2^exponent
    exponent = exponent.to(torch.int32) - 7 + (mantissa * 128 >= 127.5).to(torch.int32)
    exponent = exponent.clamp_min(least)
    out = torch.round(groups * _power(-exponent)) * _power(exponent)
    return out.view(rows, -1)[:, :features]


def _plain_norm(state):
    case, x32 = state["case"], state["x"].float()
    w32, b32 = state["weight"].float(), state["bias"].float()
    mean = x32.mean(-1, keepdim=True)
    spread = x32 - mean
    inverse = 1 / torch.sqrt(spread.square().mean(-1, keepdim=True) + EPS)
    hat = spread * inverse
    y = (hat * w32 + b32).to(state["x"].dtype)
    if not case["train"]:
        return {"y": y}
    if case["eight"]:
        centre = 0.5 * x32.amin(-1, keepdim=True) + 0.5 * x32.amax(-1, keepdim=True)
        kept = _eight(x32 - centre, LEAST_EXPONENT[torch.float32])
        hat = (kept - (mean - centre)) * inverse
    g32 = state["grad"].float()
    a = g32 * w32
    dx = inverse * (a - a.mean(-1, keepdim=True) - hat * (a * hat).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(y.dtype),
            "dweight": (g32 * hat).sum(0).to(state["weight"].dtype),
            "dbias": g32.sum(0).to(state["bias"].dtype)}


def _plain_checkpoint(state):
    x = state["x"]
    return {"read": _eight(x.float(), LEAST_EXPONENT[x.dtype]).to(x.dtype)}


def _plain_activation(state):
    x, kind = state["x"], state["case"]["kind"]
    z, g32 = x.float(), state["grad"].float()
    kept = _eight(z, LEAST_EXPONENT[x.dtype])
    if kind == "sine":
        y, slope = torch.sin(30 * z), 30 * torch.cos(30 * kept)
    elif kind == "gelu":
        y = 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
        slope = 0.5 * (1 + torch.erf(kept * math.sqrt(0.5))) + \
            kept * torch.exp(-0.5 * kept * kept) / math.sqrt(2 * math.pi)
    else:
        y = z / (1 + torch.exp(-z))
        s = 1 / (1 + torch.exp(-kept))
        slope = s * (1 + kept * (1 - s))
    return {"y": y.to(x.dtype), "dx": (g32 * slope).to(x.dtype)}


def _plain_linear(state):
    x, w32 = state["x"], state["weight"].float()
    y = (x.float() @ w32.t() + state["bias"].float()).to(x.dtype)
    if not state["case"]["train"]:
        return {"y": y}
    g32 = state["grad"].float()
    kept = _eight(x.float(), LEAST_EXPONENT[x.dtype])
    return {"y": y, "dx": (g32 @ w32).to(x.dtype), "dweight": (g32.t() @ kept).to(x.dtype),
            "dbias": g32.sum(0).to(x.dtype)}


# --------------------------------------------------------------------------
# The framework's operators


def _own_call(state):
    from diff_gabor_splatting_amd import layers

    case = state["case"]
    if case["op"] == "layer_norm":
        return layers.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS,
                                 checkpoint="8bit" if case["eight"] else "full")
    if case["op"] == "checkpoint":
        return layers.dequantize(layers.quantize(state["x"]))
    if case["op"] == "activation":
        return layers.activation(state["x"], case["kind"])
    return layers.linear(state["x"], state["weight"], state["bias"])


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"layer_norm": _plain_norm, "checkpoint": _plain_checkpoint,
                    "activation": _plain_activation, "linear": _plain_linear}[case["op"]](state)
    if case["op"] == "checkpoint":
        return {"read": _own_call(state)}
    if not case["train"]:
        with torch.no_grad():
            return {"y": _own_call(state)}
    y = _own_call(state)
    if case["op"] == "activation":
        (dx,) = torch.autograd.grad(y, (state["x"],), state["grad"])
        return {"y": y, "dx": dx}
    dx, dweight, dbias = torch.autograd.grad(
        y, (state["x"], state["weight"], state["bias"]), state["grad"])
    return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}


# --------------------------------------------------------------------------
# The operators' definition in 64 bits


def _held(values, least):
    """float64 rows as their 8-bit form stands for them, group by group of
    the row, with powers of two from a table."""
    table = torch.from_numpy(np.ldexp(1.0, np.arange(-256, 257))).to(values.device)
    out = torch.empty_like(values)
    for first in range(0, values.shape[1], GROUP):
        group = values[:, first:first + GROUP]
        largest = group.abs().max(1, keepdim=True).values
        exponent = torch.floor(torch.log2(largest.clamp_min(1e-300))).clamp(-200, 200).long() - 8
        for _ in range(3):  # up to the first exponent at which 127 holds the largest
            exponent += (torch.round(largest * table[256 - exponent]) > 127).long()
        exponent = exponent.clamp_min(least)
        out[:, first:first + GROUP] = \
            torch.round(group * table[256 - exponent]) * table[256 + exponent]
    return out


def exact(case, seed):
    state = {k: v.detach() if isinstance(v, torch.Tensor) else v
             for k, v in prepare(case, seed).items()}
    least = LEAST_EXPONENT[state["x"].dtype]
    x = state["x"].double()
    if case["op"] == "checkpoint":
        return {"read": _held(x, least)}
    g = state["grad"].double() if case["train"] else None
    if case["op"] == "activation":
        k = _held(x, least)
        if case["kind"] == "sine":
            return {"y": torch.sin(30 * x), "dx": g * 30 * torch.cos(30 * k)}
        if case["kind"] == "gelu":
            return {"y": x * torch.special.ndtr(x),
                    "dx": g * (torch.special.ndtr(k)
                               + k * torch.exp(-k * k / 2) / math.sqrt(2 * math.pi))}
        s = torch.sigmoid(k)
        return {"y": x * torch.sigmoid(x), "dx": g * (s + k * s * (1 - s))}
    w, b = state["weight"].double(), state["bias"].double()
    if case["op"] == "linear":
        y = torch.addmm(b, x, w.t())
        if not case["train"]:
            return {"y": y}
        return {"y": y, "dx": torch.mm(g, w), "dweight": torch.mm(g.t(), _held(x, least)),
                "dbias": g.sum(0)}
    variance, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    deviation = torch.sqrt(variance + EPS)
    y = (x - mean) / deviation * w + b
    if not case["train"]:
        return {"y": y}
    if case["eight"]:
        # What is kept is a float32 difference from a float32 centre.
        low, high = torch.aminmax(state["x"].float(), dim=1, keepdim=True)
        centre = ((low.double() + high.double()) / 2).float()
        x = centre.double() + _held((state["x"].float() - centre).double(), -126)
    h = (x - mean) / deviation
    h_sum, a_sum = (g * w * h).mean(1, keepdim=True), (g * w).mean(1, keepdim=True)
    return {"y": y, "dx": (g * w - a_sum - h * h_sum) / deviation,
            "dweight": (g * h).sum(0), "dbias": g.sum(0)}
