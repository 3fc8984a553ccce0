"""The decoder layers in 64 bits, by their formulas (see gabor_layers.h).

Everything is float64 on the CPU; ``kept`` is the 8-bit form, given as its
bytes, its exponent bytes and the values that they stand for.
"""

from __future__ import annotations

import math

import numpy as np
import torch

GROUP = 32
LIMITS = {torch.float32: (1, 248), torch.bfloat16: (1, 248), torch.float16: (103, 136)}


def kept(x: torch.Tensor, dtype=None):
    """(bytes int8 [rows, 32 G], exponents uint8 [rows, G], values float64) of
    rows ``x``; ``dtype`` (default: that of x) sets the exponents' range."""
    least, most = LIMITS[dtype or x.dtype]
    rows, features = x.shape
    groups = -(-features // GROUP)
    values = np.zeros((rows, groups * GROUP))
    values[:, :features] = x.double().numpy()
    values = values.reshape(rows, groups, GROUP)
    fine = np.isfinite(values).all(-1)
    held = np.where(fine[..., None], values, 0.0)
    largest = np.abs(held).max(-1)
    exponents = np.full((rows, groups), least)
    for _ in range(most - least):  # the definition: the first that is enough
        short = (np.rint(np.ldexp(largest, 127 - exponents)) > 127) & (exponents < most)
        if not short.any():
            break
        exponents = exponents + short
    q = np.clip(np.rint(np.ldexp(held, 127 - exponents[..., None])), -127, 127)
    stands = np.ldexp(q, exponents[..., None] - 127)
    stands[~fine] = np.nan
    exponents[~fine] = 255
    return (torch.from_numpy(q.astype(np.int8)).reshape(rows, -1),
            torch.from_numpy(exponents.astype(np.uint8)),
            torch.from_numpy(stands).reshape(rows, -1)[:, :features])


def _phi(z):
    return torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def activation(z: torch.Tensor, kind: str, omega: float) -> torch.Tensor:
    z = z.double()
    if kind == "sine":
        return torch.sin(omega * z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(z)


def slope(z: torch.Tensor, kind: str, omega: float) -> torch.Tensor:
    z = z.double()
    if kind == "sine":
        return omega * torch.cos(omega * z)
    if kind == "gelu":
        return torch.special.ndtr(z) + z * _phi(z)
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


def centre(x: torch.Tensor) -> torch.Tensor:
    """The middle of each row's range, as float32 arithmetic gives it."""
    x = x.float()
    return 0.5 * x.amin(1, keepdim=True) + 0.5 * x.amax(1, keepdim=True)


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5):
    """(y, normalised rows h, inverse deviation r)."""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    h = (x - mean) * r
    y = h if weight is None else h * weight.double()
    return (y if bias is None else y + bias.double()), h, r


def layer_norm_backward(x, grad, weight=None, eps: float = 1e-5, eight: bool = False):
    """(dx, dweight, dbias, h as the backward pass has it, r)."""
    _, h, r = layer_norm(x, eps=eps)
    if eight:
        c = centre(x)
        d = kept(x.float() - c, torch.float32)[2]
        h = (d - (x.double().mean(1, keepdim=True) - c.double())) * r
    g = grad.double()
    a = g if weight is None else g * weight.double()
    dx = r * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    return dx, (g * h).sum(0), g.sum(0), h, r


def linear(x, weight, bias=None):
    y = x.double() @ weight.double().t()
    return y if bias is None else y + bias.double()


def linear_backward(x, weight, grad):
    """(dx, dweight, dbias)."""
    g = grad.double()
    return g @ weight.double(), g.t() @ kept(x)[2], g.sum(0)
