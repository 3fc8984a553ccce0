"""Layers of a surfel decoder: what turns a latent vector per surfel into the
values that the renderers take.

``layer_norm``, ``linear`` and ``activation`` work on rows of features (any
leading dimensions) in float32, bfloat16 or float16 on a HIP device, with
first-order reverse-mode autograd (forward mode and tracing are refused). Over
a scene's surfels it is the activations kept for the backward pass that fill
memory, so these keep them in 8 bits: 33/32 bytes a value instead of two or
four.

The 8-bit form (:class:`Checkpoint`, :func:`quantize`, :func:`dequantize`):
each 32 consecutive features of a row share a power of two, the smallest with
which the largest of them rounds to at most 127, and each is kept as the
nearest integer multiple of it (ties to even). The error of a value is at most
1/127 of the largest of its group (half a step; a power of two, because then a
kept value is exact in the type it came from and does not depend on how a scale
was rounded). A group with an infinity or a NaN reads back as NaN.

All work is queued on the current stream; nothing synchronises. Inputs whose
features are contiguous and whose leading dimensions collapse are read in
place, others are copied first. ``include/gabor_layers.h`` has the C entry
points.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import _native

_host = _native._host

GROUP = 32
ACTIVATIONS = {"sine": 0, "gelu": 1, "silu": 2}
_CHECKPOINTS = {"full": False, "8bit": True}

__all__ = ["Checkpoint", "quantize", "dequantize", "activation", "layer_norm", "linear"]


class Checkpoint:
    """A tensor in 8 bits: ``values`` int8 [rows, 32 G] and ``exponents`` uint8
    [rows, G], G = ceil(features / 32); value = q 2^(exponent - 127). ``shape``
    and ``dtype`` are those of the tensor it was made from."""

    __slots__ = ("values", "exponents", "shape", "dtype")

    def __init__(self, values: Tensor, exponents: Tensor, shape, dtype: torch.dtype):
        self.values, self.exponents = values, exponents
        self.shape, self.dtype = torch.Size(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.values.nbytes + self.exponents.nbytes

    def __repr__(self) -> str:
        return f"Checkpoint(shape={tuple(self.shape)}, dtype={self.dtype}, nbytes={self.nbytes})"


def _tensor(name: str, value) -> Tensor:
    if not isinstance(value, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    return value


def _number(name: str, value) -> None:
    # A learned one would be read here and never get its gradient.
    if isinstance(value, Tensor) and value.requires_grad:
        raise ValueError(f"{name} has no gradient: pass a number, or a detached tensor")


def quantize(x: Tensor) -> Checkpoint:
    """``x`` in 8 bits, in groups of 32 features. Not differentiable."""
    values, exponents = _host.checkpoint8_write(_tensor("x", x))
    return Checkpoint(values, exponents, x.shape, x.dtype)


def dequantize(checkpoint: Checkpoint, dtype: Optional[torch.dtype] = None) -> Tensor:
    """What the checkpoint stands for, contiguous, in the type it was made from
    or in ``dtype`` (float16 of another type's is rounded where it has no such
    value)."""
    if not isinstance(checkpoint, Checkpoint):
        raise TypeError("checkpoint must be a Checkpoint")
    return _host.checkpoint8_read(checkpoint.values, checkpoint.exponents,
                                  list(checkpoint.shape), dtype or checkpoint.dtype)


def activation(x: Tensor, kind: str = "sine", omega: float = 30.0) -> Tensor:
    """``sin(omega x)`` (the neural renderer's, "sine"), ``x Phi(x)`` ("gelu")
    or ``x / (1 + exp(-x))`` ("silu"). The backward pass takes the derivative
    at the input as kept in 8 bits."""
    if kind not in ACTIVATIONS:
        raise ValueError(f"kind must be one of {', '.join(map(repr, ACTIVATIONS))}")
    _number("omega", omega)
    if not math.isfinite(omega):
        raise ValueError("omega must be finite")
    return _host.activation(_tensor("x", x), ACTIVATIONS[kind], omega)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, checkpoint: str = "full") -> Tensor:
    """Layer norm over the last dimension (at most 16384 features): ``(x - mean)
    / sqrt(variance + eps) * weight + bias``. ``weight`` and ``bias`` are
    [features] in the type of ``x`` or in float32, or None. The backward pass
    reads ``x`` itself ("full") or ``x`` less the middle of its row's range,
    kept in 8 bits ("8bit")."""
    if checkpoint not in _CHECKPOINTS:
        raise ValueError("checkpoint must be 'full' or '8bit'")
    _number("eps", eps)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    return _host.layer_norm(_tensor("x", x), weight, bias, eps, _CHECKPOINTS[checkpoint])


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    """``x weight^T + bias`` with ``weight`` [outputs, features], all of one
    type. The weight's gradient is taken with the input as kept in 8 bits; the
    input's gradient does not depend on it."""
    return _host.linear(_tensor("x", x), _tensor("weight", weight), bias)
