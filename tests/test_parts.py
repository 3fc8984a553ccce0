"""Rows in groups, layers by group and dropout against their formulas in 64
bits (oracle/parts.py).

CPU: the oracle's generator against its published answers, argument errors
of the C entry points and of the Python functions. GPU: every operator over
types, sizes, groups and layouts.

Tolerances are worst-case rounding bounds, as in test_layers.py: with u the
unit roundoff of the output type and e = 2^-24, an output that is computed in
float32 and rounded once is off by at most u |out| + the float32 error, and a
float32 sum of n terms t by at most n e sum |t|.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import parts as oracle
from test_layers import DTYPES, E, gpu_test, layers, near, normal

# --------------------------------------------------------------------------
# CPU


@pytest.mark.parametrize("counter,key,answer", [
    ([0] * 4, [0] * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     "d16cfe09 94fdcceb 5001e420 24126ea1")])
def test_oracle_generator_gives_the_published_answers(counter, key, answer):
    words = oracle.philox(np.array([counter], dtype=np.uint64), key)[0]
    assert " ".join(f"{w:08x}" for w in words) == answer


def test_oracle_groups():
    order, offsets = oracle.row_groups(torch.tensor([2, -1, 0, 2, 7, 0]), 3)
    assert order.tolist() == [2, 5, 0, 3, 1, 4] and offsets.tolist() == [0, 2, 2, 4]


def refused(lib, status, code, text):
    assert status == code and text in lib.gs_last_error().decode(), lib.gs_last_error()


def test_c_entry_points_refuse_bad_arguments():
    from diff_gabor_splatting_amd import _native

    lib, p = _native.lib, ctypes.c_void_p(256)
    refused(lib, lib.gs_dropout(3, 0.5, 0, None, p, 8, 1, 8, p, None), 1, "unknown type")
    refused(lib, lib.gs_dropout(0, 1.5, 0, None, p, 8, 1, 8, p, None), 1, "0 through 1")
    refused(lib, lib.gs_dropout(0, math.nan, 0, None, p, 8, 1, 8, p, None), 1, "0 through 1")
    refused(lib, lib.gs_dropout(0, 0.5, 0, None, p, 7, 2, 8, p, None), 1, "overlap")
    refused(lib, lib.gs_dropout(0, 0.5, 0, None, None, 8, 1, 8, p, None), 1, "null")
    refused(lib, lib.gs_dropout(0, 0.5, 0, None, p, 8, 1 << 33, 8, p, None), 2, "too many rows")
    assert lib.gs_dropout(0, 0.5, 0, None, None, 8, 0, 8, None, None) == 0
    refused(lib, lib.gs_row_groups(0, p, -1, 4, p, p, None, 0, None), 2, "rows")
    refused(lib, lib.gs_row_groups(0, p, 1 << 31, 4, p, p, None, 0, None), 2, "rows")
    refused(lib, lib.gs_row_groups(0, p, 8, 0, p, p, None, 0, None), 1, "groups")
    refused(lib, lib.gs_row_groups(0, p, 8, 4097, p, p, None, 0, None), 1, "groups")
    refused(lib, lib.gs_row_groups(0, p, 8, 4, None, p, None, 0, None), 1, "null")
    need = lib.gs_row_groups_workspace_size(100_000, 64)
    assert need > 0
    refused(lib, lib.gs_row_groups(0, p, 100_000, 64, p, p, p, need - 1, None), 4, "workspace")


def test_python_functions_refuse_bad_arguments():
    m = layers()
    x = torch.zeros(2, 8)
    for call in (lambda: m.dropout(x), lambda: m.row_groups(torch.zeros(4, dtype=torch.int32), 2)):
        with pytest.raises(ValueError, match="on a HIP device"):
            call()
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        m.dropout([1.0])
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="p must be"):
            m.dropout(x, p)
    with pytest.raises(ValueError, match="p has no gradient"):
        m.dropout(x, torch.tensor(0.5, requires_grad=True))
    with pytest.raises(ValueError, match="64 bits"):
        m.dropout(x, 0.5, 1 << 64)
    with pytest.raises(TypeError):
        m.dropout(x, 0.5, 1.5)
    with pytest.raises(TypeError, match="index must be"):
        m.row_groups([0, 1], 2)
    for groups in (0, 4097):
        with pytest.raises(ValueError, match="groups must be"):
            m.row_groups(torch.zeros(4, dtype=torch.int32), groups)
    offsets, order = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for bad in (offsets.long(), offsets[:1], offsets[None], torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="offsets must be"):
            m.RowGroups(bad, order)
    for bad in (order.long(), order[None], torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="order must be"):
            m.RowGroups(offsets, bad)
    assert m.RowGroups(offsets, order).groups == 2
    assert repr(m.RowGroups(offsets, order)) == "RowGroups(groups=2, rows=4)"


# --------------------------------------------------------------------------
# GPU: dropout


def check_dropout(x, g, p, seed, y, dx):
    """One rounding of the scale, one of the product in float32, one to the type."""
    rows, features = x.numel() // x.shape[-1], x.shape[-1]
    for got, from_ in ((y, x), (dx, g)):
        want = oracle.dropout(from_.reshape(rows, features), p, seed)
        near(got.reshape(rows, features), want, 2 * E * want.abs(), x.dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 57), (2, 3, 40), (64,), (1000, 187),
                                   (300, 1024), (40_000, 96), (30_001, 100)])
def test_dropout(dtype, shape):
    m = layers()
    x, g = normal(*shape, seed=1, dtype=dtype), normal(*shape, seed=2, dtype=dtype)
    on = x.cuda().requires_grad_()
    y = m.dropout(on, 0.3, 1234567890123)
    (dx,) = torch.autograd.grad(y, on, g.cuda())
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    check_dropout(x, g, 0.3, 1234567890123, y, dx)
    with torch.no_grad():
        assert torch.equal(m.dropout(on, 0.3, 1234567890123), y)


@gpu_test
@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1 - 2.0 ** -18,
                               1.0])
def test_dropout_of_every_share(p):
    m = layers()
    x, g = normal(500, 200, seed=3), normal(500, 200, seed=4)
    on = x.cuda().requires_grad_()
    y = m.dropout(on, p, 5)
    check_dropout(x, g, p, 5, y, torch.autograd.grad(y, on, g.cuda())[0])
    if p in (0.0, 2.0 ** -18):
        assert torch.equal(y.cpu(), x)
    if p in (1.0, 1 - 2.0 ** -18):
        assert not y.any()


@gpu_test
@pytest.mark.parametrize("seed", [0, 1, -1, -(1 << 63), (1 << 64) - 1, 1 << 63, 0xFFFFFFFF00000001])
def test_dropout_seeds(seed):
    m = layers()
    x = normal(70, 64, seed=6)
    y = m.dropout(x.cuda(), 0.5, seed)
    near(y, oracle.dropout(x, 0.5, seed), 2 * E * x.double().abs() * 2, torch.float32)
    if -(1 << 63) <= seed < 1 << 63:
        word = torch.tensor([seed], device="cuda")
        assert torch.equal(m.dropout(x.cuda(), 0.5, word), y)


@gpu_test
def test_dropout_drops_bad_values_and_keeps_the_rest():
    m = layers()
    x = normal(64, 64, seed=7)
    keep = oracle.dropout_bits(range(64), 64, 9) >= 32768
    bad = torch.where(keep, x, torch.tensor([math.nan, math.inf] * 32))
    assert torch.equal(m.dropout(bad.cuda(), 0.5, 9), m.dropout(x.cuda(), 0.5, 9))
    assert not torch.signbit(m.dropout(bad.cuda(), 0.5, 9).cpu()[~keep]).any()
    kept = torch.where(keep, math.inf, x)
    assert torch.equal(m.dropout(kept.cuda(), 0.5, 9).cpu().isinf(), keep)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_of_strided_rows(dtype):
    m = layers()
    base = normal(12, 4, 200, seed=8, dtype=dtype).cuda()
    for view in (lambda t: t[:, 1, :96], lambda t: t[:, 2, 3:100], lambda t: t[:, :3, 8:72],
                 lambda t: t.transpose(0, 2), lambda t: t[:1, 0, :40].expand(6, 40),
                 lambda t: t[:, :, :1], lambda t: t[:, 0, ::2]):
        x = view(base)
        assert torch.equal(m.dropout(x, 0.4, 3), m.dropout(x.contiguous(), 0.4, 3))


@gpu_test
def test_dropout_of_no_rows():
    m = layers()
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = m.dropout(x)
    assert y.shape == (0, 8) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 8)


@gpu_test
def test_dropout_in_a_graph_draws_from_its_seed():
    """A replayed graph takes the seed that its word holds then."""
    m = layers()
    x = normal(3000, 64, seed=10).cuda().requires_grad_()
    g = normal(3000, 64, seed=11).cuda()
    word = torch.tensor([1], device="cuda")

    def step():
        y = m.dropout(x, 0.3, word)
        return y, torch.autograd.grad(y, x, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6, 5):
        word.fill_(seed)
        graph.replay()
        torch.cuda.synchronize()
        y = m.dropout(x, 0.3, seed)
        want = (y, torch.autograd.grad(y, x, g)[0])
        for got, expected in zip(out, want):
            assert torch.equal(got, expected)


@gpu_test
def test_dropout_seed_may_not_change_before_the_backward_pass():
    m = layers()
    x, word = torch.ones(4, 8, device="cuda", requires_grad=True), torch.tensor([1], device="cuda")
    y = m.dropout(x, 0.5, word)
    word.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# --------------------------------------------------------------------------
# GPU: rows in groups


@gpu_test
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,groups", [(1, 1), (5, 3), (64, 2), (65, 64), (1023, 7), (1024, 4096),
                                         (1025, 65), (5000, 1), (60_000, 255), (60_000, 4096),
                                         (262_145, 100), (300_000, 512)])
def test_row_groups(kind, rows, groups):
    m = layers()
    gen = torch.Generator().manual_seed(rows + groups)
    index = torch.randint(-1, groups + 1, (rows,), generator=gen)
    if rows > 100:  # a long run of one group, some groups without a row
        index[20:90] = 0
        index[index == groups // 2] = -7
    index[::97] = torch.iinfo(kind).max
    index[5::97] = torch.iinfo(kind).min
    got = m.row_groups(index.to(kind).cuda(), groups)
    order, offsets = oracle.row_groups(index, groups)
    assert torch.equal(got.offsets.cpu(), offsets) and torch.equal(got.order.cpu(), order)


@gpu_test
def test_row_groups_of_any_shape():
    m = layers()
    index = torch.randint(0, 5, (6, 70), generator=torch.Generator().manual_seed(1))
    for view in (index, index.t(), index[:, ::3], index[:0]):
        got = m.row_groups(view.cuda(), 5)
        order, offsets = oracle.row_groups(view, 5)
        assert torch.equal(got.offsets.cpu(), offsets) and torch.equal(got.order.cpu(), order)


@gpu_test
def test_row_groups_refuse_other_types():
    m = layers()
    for bad in (torch.float32, torch.int16, torch.uint8, torch.bool):
        with pytest.raises(ValueError, match="int32 or int64"):
            m.row_groups(torch.zeros(4, device="cuda").to(bad), 2)


@gpu_test
def test_dropout_seed_refusals():
    m = layers()
    x = torch.zeros(2, 8, device="cuda")
    for bad in (torch.tensor([1]), torch.tensor([1], dtype=torch.int32, device="cuda"),
                torch.tensor([1, 2], device="cuda")):
        with pytest.raises(ValueError, match="seed must be"):
            m.dropout(x, 0.5, bad)
