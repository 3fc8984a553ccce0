"""Layers by group at their edges: infinities, scales far from one, gradients
asked for alone, the widest tiles and the joins of many parts, groups that
change under a captured graph, and memory beside the results.

Tolerances as in test_parts.py.
"""

import math

import pytest
import torch

from oracle import parts as oracle
from test_layers import DTYPES, E, gpu_test, layers, near, normal
from test_parts import INNER, grouped_by

# --------------------------------------------------------------------------
# Infinities


def positive(*shape, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    return (0.5 + torch.rand(shape, generator=gen)).to(dtype)


INFINITE_CASES = pytest.mark.parametrize("rows,features,rank", [
    (rows, *size) for rows in (9, 300)
    for size in ((40, 1), (40, 5), (40, 31), (40, 32), (40, 33), (40, 63), (1100, 5), (1100, 40))])


def infinite_rows(dtype, rows, features, rank):
    """(y, dx, da, du) and what the formula gives, all values positive: an
    infinity wherever one is met, and never a NaN. Wide rows go by tiles, the
    others by streaming. One inner row is whole numbers."""
    m = layers()
    outputs, groups, scale = 24, 3, 0.5
    by, members = grouped_by(torch.arange(rows) % 4 - 1, groups)
    x, w = positive(rows, features, seed=1, dtype=dtype), positive(outputs, features, seed=2,
                                                                 dtype=dtype)
    a = torch.ones(groups, rank, features, dtype=dtype)
    u, g = positive(groups, outputs, rank, seed=3, dtype=dtype), positive(rows, outputs, seed=4,
                                                                        dtype=dtype)
    x[5, 3], x[6], g[6, 7], x[4, 2], g[8, 1] = math.inf, 1, math.inf, math.inf, math.inf
    on, ac, uc = (t.cuda().requires_grad_() for t in (x, a, u))
    y = m.adapted_linear(on, w.cuda(), ac, uc, by, scale=scale)
    got = (y, *torch.autograd.grad(y, (on, ac, uc), g.cuda()))
    want = oracle.adapted_linear(x, w, a, u, members, None, scale, g)
    most = max(len(at) for at in members)
    # All terms are positive, so sums are their own sums of magnitudes; float16's
    # parts go by the row's largest value, within a factor of 9 of any other.
    error = (features + outputs + rank + most + 8) * 2 * E + 9 * INNER[dtype]
    return list(zip(got, want)), error


def infinite_where_expected(got, expected, error, dtype):
    got = got.detach().cpu()
    assert not expected.isnan().any() and not got.isnan().any()
    assert torch.equal(got.isinf(), expected.isinf()) and (got[got.isinf()] > 0).all()
    fine = expected.isfinite()
    near(got[fine], expected[fine], error * expected[fine], dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@INFINITE_CASES
def test_adapted_linear_of_rows_with_infinities(dtype, rows, features, rank):
    results, error = infinite_rows(dtype, rows, features, rank)
    for got, expected in results[:2]:
        infinite_where_expected(got, expected, error, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@INFINITE_CASES
def test_adapters_gradients_of_rows_with_infinities(dtype, rows, features, rank):
    results, error = infinite_rows(dtype, rows, features, rank)
    for got, expected in results[2:]:
        infinite_where_expected(got, expected, error, dtype)
