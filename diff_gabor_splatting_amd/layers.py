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

Surfels that belong to parts go through ``grouped_linear`` (a matrix to each
group of rows) or ``adapted_linear`` (a shared matrix, a low-rank adapter to
each group) by the :class:`RowGroups` that :func:`row_groups` makes; these keep
their input whole. ``dropout`` keeps nothing.

All work is queued on the current stream; nothing synchronises. Inputs whose
features are contiguous and whose leading dimensions collapse are read in
place, others are copied first. ``include/gabor_layers.h`` has the C entry
points.
"""

from __future__ import annotations

import math
import operator
from typing import Optional, Union

import torch
from torch import Tensor

from . import _native

_host = _native._host

GROUP = 32
ACTIVATIONS = {"sine": 0, "gelu": 1, "silu": 2}
_CHECKPOINTS = {"full": False, "8bit": True}

__all__ = ["Checkpoint", "quantize", "dequantize", "activation", "layer_norm", "linear", "dropout",
           "RowGroups", "row_groups", "grouped_linear", "adapted_linear"]


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
    other gradients do not depend on it."""
    return _host.linear(_tensor("x", x), _tensor("weight", weight), bias)


def dropout(x: Tensor, p: float = 0.5, seed: Union[int, Tensor] = 0) -> Tensor:
    """``x / (1 - p)`` where a mask keeps a value, 0 where it does not (a NaN
    that is dropped, too). Nothing is kept for the backward pass: the mask is
    a function of ``seed`` and of a value's row and column (the leading
    dimensions counted as one), from a counter-based generator
    (Philox4x32-10; ``include/gabor_layers.h`` has the definition). The same
    seed gives the same mask, so a program takes another for each layer and
    step. ``seed`` is a 64-bit integer, or one int64 on the device of ``x``,
    which is read when the call runs, in a replayed HIP graph too; it may not
    change between the forward and the backward pass. ``p`` is rounded to a multiple
    of 2^-16, and 1 / (1 - p) is that of the rounded one."""
    _tensor("x", x)
    _number("p", p)
    if not 0 <= p <= 1:  # not for a NaN, either
        raise ValueError("p must be 0 through 1")
    if isinstance(seed, Tensor):
        return _host.dropout(x, p, 0, seed)
    seed = operator.index(seed)
    if not -(1 << 63) <= seed < 1 << 64:
        raise ValueError("seed must fit 64 bits")
    return _host.dropout(x, p, (seed + (1 << 63)) % (1 << 64) - (1 << 63), None)


class RowGroups:
    """Rows that belong to groups: ``offsets`` int32 [groups + 1], not falling,
    and ``order`` int32 [rows], a permutation of the rows: the rows of group g
    are ``order[offsets[g]:offsets[g + 1]]``, those at other places of ``order``
    are in no group. Without an order the rows lie by group themselves.
    :func:`row_groups` makes one of each row's group."""

    __slots__ = ("offsets", "order")

    def __init__(self, offsets: Tensor, order: Optional[Tensor] = None):
        _tensor("offsets", offsets)
        if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 2 or \
                not offsets.is_contiguous():
            raise ValueError("offsets must be contiguous int32 of shape (groups + 1,)")
        if order is not None:
            _tensor("order", order)
            if order.dtype != torch.int32 or order.dim() != 1 or not order.is_contiguous():
                raise ValueError("order must be contiguous int32 of shape (rows,)")
            if order.device != offsets.device:
                raise ValueError("order must be on the device of offsets")
        self.offsets, self.order = offsets, order

    @property
    def groups(self) -> int:
        return self.offsets.numel() - 1

    def __repr__(self) -> str:
        rows = "" if self.order is None else f", rows={self.order.numel()}"
        return f"RowGroups(groups={self.groups}{rows})"


def row_groups(index: Tensor, groups: int) -> RowGroups:
    """The rows by group: ``index`` (int32 or int64, any shape) is each row's
    group, 0 through ``groups - 1``, and any other number puts a row in none.
    Rows keep their order within a group. At most 4096 groups and 2^31 - 4096
    rows."""
    groups = operator.index(groups)
    if not 1 <= groups <= 4096:
        raise ValueError("groups must be 1 through 4096")
    return RowGroups(*_host.row_groups(_tensor("index", index), groups))


def _groups(groups) -> RowGroups:
    if not isinstance(groups, RowGroups):
        raise TypeError("groups must be a RowGroups")
    return groups


def grouped_linear(x: Tensor, weight: Tensor, groups: RowGroups,
                   bias: Optional[Tensor] = None) -> Tensor:
    """``x weight[g]^T + bias[g]`` for the rows of group g, 0 for rows of no
    group (whose gradient is 0, too). ``weight`` [groups, outputs, features]
    and ``bias`` [groups, outputs] have the type of ``x``. Rows are read and
    written where they lie. The backward pass reads ``x`` itself, for the
    matrices' gradients."""
    groups = _groups(groups)
    return _host.grouped_linear(_tensor("x", x), _tensor("weight", weight), groups.offsets,
                                groups.order, bias)


def adapted_linear(x: Tensor, weight: Tensor, down: Tensor, up: Tensor, groups: RowGroups,
                   bias: Optional[Tensor] = None, scale: float = 1.0) -> Tensor:
    """``x weight^T + bias + scale (x down[g]^T) up[g]^T`` for the rows of group
    g, without the last term for rows of no group: a linear layer that all rows
    share, with an adapter of each row's group beside it. ``weight``
    [outputs, features], ``bias`` [outputs], ``down`` [groups, rank, features]
    and ``up`` [groups, outputs, rank] have the type of ``x``; the rank is at
    most 64. The backward pass reads ``x`` itself for the adapters' gradients, and
    the shared matrix's gradient is that of :func:`linear`, taken with the
    input in 8 bits; none is computed that is not asked for. An infinity in an
    adapter's matrix may give NaN where the formula has an infinity."""
    groups = _groups(groups)
    _number("scale", scale)
    # As the kernels take it: a larger number is an infinity there.
    if not math.isfinite(scale) or abs(scale) > 3.4e38:
        raise ValueError("scale must be finite in float32")
    return _host.adapted_linear(_tensor("x", x), _tensor("weight", weight),
                                _tensor("down", down), _tensor("up", up), groups.offsets,
                                groups.order, bias, scale)
