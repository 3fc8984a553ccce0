"""Rows in groups, layers by group and dropout in 64 bits, by their
formulas (see gabor_layers.h). Everything is float64 on the CPU."""

from __future__ import annotations

import numpy as np
import torch


def philox(counter, key):
    """Philox4x32-10 of uint32 words: counter [..., 4], key (2,)."""
    c = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    word = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        half = np.uint64(32)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & word,
             (a >> half) ^ c[3] ^ np.uint64(k[1]), a & word]
        k = [(k[0] + 0x9E3779B9) % (1 << 32), (k[1] + 0xBB67AE85) % (1 << 32)]
    return np.stack(c, -1).astype(np.uint32)


def dropout_bits(rows, features: int, seed: int) -> torch.Tensor:
    """The 16 bits of each value of the given rows (numbers)."""
    rows = np.asarray(rows, dtype=np.uint64)
    chunks = -(-features // 8)
    counter = np.zeros((len(rows), chunks, 4), dtype=np.uint64)
    counter[..., 0] = np.arange(chunks, dtype=np.uint64)
    counter[..., 1] = (rows & np.uint64(0xFFFFFFFF))[:, None]
    counter[..., 2] = (rows >> np.uint64(32))[:, None]
    seed %= 1 << 64
    words = philox(counter, (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack((words & 0xFFFF, words >> 16), -1).reshape(len(rows), chunks * 8)
    return torch.from_numpy(halves[:, :features].astype(np.int64))


def dropout(x: torch.Tensor, p: float, seed: int, rows=None) -> torch.Tensor:
    """Rows ``x`` (numbered ``rows``, 0 on by default) through the mask."""
    least = round(65536 * p)
    keep = dropout_bits(range(len(x)) if rows is None else rows, x.shape[1], seed) >= least
    scale = 65536 / (65536 - least) if least < 65536 else 0.0
    return torch.where(keep, x.double() * scale, 0.0)


def row_groups(index: torch.Tensor, groups: int):
    """(order, offsets) of each row's group."""
    index = index.reshape(-1).tolist()
    members = [[] for _ in range(groups + 1)]
    for row, group in enumerate(index):
        members[group if 0 <= group < groups else groups].append(row)
    offsets = np.cumsum([0] + [len(m) for m in members[:-1]])
    order = [row for m in members for row in m]
    return torch.tensor(order, dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32)


def members(offsets, order, rows: int):
    """The rows of each group, as tensors."""
    order = torch.arange(rows) if order is None else order.long().cpu()
    at = offsets.long().cpu().tolist()
    return [order[a:b] for a, b in zip(at[:-1], at[1:])]


def grouped_linear(x, weight, groups, bias=None, grad=None):
    """y, and with ``grad`` also (dx, dweight, dbias); ``groups`` as
    :func:`members` gives them. A row of no group has y = dx = 0."""
    x, weight = x.double(), weight.double()
    y = x.new_zeros(len(x), weight.shape[1])
    out = [torch.zeros_like(x), torch.zeros_like(weight), weight.new_zeros(weight.shape[:2])]
    for g, rows in enumerate(groups):
        y[rows] = x[rows] @ weight[g].t()
        if bias is not None:
            y[rows] += bias[g].double()
        if grad is not None:
            d = grad.double()[rows]
            out[0][rows] = d @ weight[g]
            out[1][g] = d.t() @ x[rows]
            out[2][g] = d.sum(0)
    return y if grad is None else (y, *out)


def adapted_linear(x, weight, down, up, groups, bias=None, scale=1.0, grad=None):
    """y, and with ``grad`` also (dx, ddown, dup)."""
    x, weight, down, up = x.double(), weight.double(), down.double(), up.double()
    y = x @ weight.t()
    if bias is not None:
        y += bias.double()
    out = [None, torch.zeros_like(down), torch.zeros_like(up)]
    if grad is not None:
        out[0] = grad.double() @ weight
    for g, rows in enumerate(groups):
        inner = x[rows] @ down[g].t()
        y[rows] += scale * inner @ up[g].t()
        if grad is not None:
            d = grad.double()[rows]
            back = d @ up[g]
            out[0][rows] += scale * back @ down[g]
            out[1][g] = scale * back.t() @ x[rows]
            out[2][g] = scale * d.t() @ inner
    return y if grad is None else (y, *out)
