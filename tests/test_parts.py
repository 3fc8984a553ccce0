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


# --------------------------------------------------------------------------
# GPU: layers by group


def some_groups(rows, groups, seed, none=0.05, empty=True):
    """Each row's group, sizes uneven, some groups empty, some rows in none."""
    gen = torch.Generator().manual_seed(seed)
    shares = torch.rand(groups, generator=gen) ** 3 + 1e-3
    if empty and groups > 2:
        shares[::3] = 0
    index = torch.multinomial(shares, rows, replacement=True, generator=gen)
    index[torch.rand(rows, generator=gen) < none] = -1
    return index


def grouped_by(index, groups):
    """(the framework's groups, each group's rows)."""
    got = layers().row_groups(index.cuda(), groups)
    return got, oracle.members(got.offsets, got.order, index.numel())


def check_grouped(x, w, b, g, members, y, grads):
    rows, features, outputs = len(x), x.shape[1], w.shape[1]
    want = oracle.grouped_linear(x, w, members, b, g)
    size = oracle.grouped_linear(x.abs(), w.abs(), members, None if b is None else b.abs(),
                                 g.abs())
    most = max([len(m) for m in members] + [1])
    near(y.reshape(rows, outputs), want[0], (features + 2) * E * size[0], x.dtype)
    near(grads[0].reshape(rows, features), want[1], (outputs + 2) * E * size[1], x.dtype)
    near(grads[1], want[2], (most + 2) * E * size[2], x.dtype)
    if b is not None:
        near(grads[2], want[3], (most + 2) * E * size[3], x.dtype)


def grouped_case(rows, features, outputs, groups, dtype, bias=True, seed=21, index=None):
    m = layers()
    x = normal(rows, features, seed=seed, dtype=dtype)
    w = normal(groups, outputs, features, seed=seed + 1, dtype=dtype, scale=features ** -0.5)
    b = normal(groups, outputs, seed=seed + 2, dtype=dtype) if bias else None
    g = normal(rows, outputs, seed=seed + 3, dtype=dtype)
    index = some_groups(rows, groups, seed) if index is None else index
    by, members = grouped_by(index, groups)
    inputs = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    y = m.grouped_linear(inputs[0], inputs[1], by, *inputs[2:])
    grads = torch.autograd.grad(y, inputs, g.cuda())
    with torch.no_grad():
        assert torch.equal(m.grouped_linear(inputs[0], inputs[1], by, *inputs[2:]), y)
    check_grouped(x, w, b, g, members, y, grads)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs,groups", [
    (1, 1, 1, 1), (1, 1024, 57, 8), (4, 64, 64, 8), (16, 33, 18, 3), (17, 8, 8, 5), (40, 5, 3, 2),
    (64, 96, 57, 64), (127, 130, 63, 4), (300, 187, 18, 7), (1000, 40, 72, 300),
    (2500, 264, 136, 6), (1024, 64, 57, 16), (5000, 128, 128, 12), (3000, 260, 300, 2),
    (200, 1100, 40, 3), (200, 40, 1100, 3), (90, 1030, 1030, 2), (700, 512, 512, 5)])
def test_grouped_linear(dtype, rows, features, outputs, groups):
    grouped_case(rows, features, outputs, groups, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_without_bias_and_of_special_groups(dtype):
    grouped_case(500, 64, 40, 5, dtype, bias=False)
    none = torch.full((200,), -1)
    grouped_case(200, 64, 40, 5, dtype, index=none)           # no row has a group
    grouped_case(200, 64, 40, 5, dtype, index=none + 4)       # one has all
    grouped_case(3000, 64, 40, 5, dtype, index=torch.arange(3000) % 5)
    grouped_case(130, 64, 40, 130, dtype, index=torch.arange(130))  # a row each
    grouped_case(2000, 24, 8, 3000, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_of_rows_that_lie_by_group(dtype):
    """No order; rows of no group before the first group and behind the last."""
    m = layers()
    rows, features, outputs = 700, 48, 40
    offsets = torch.tensor([30, 30, 200, 455, 455, 690], dtype=torch.int32)
    x, g = normal(rows, features, seed=1, dtype=dtype), normal(rows, outputs, seed=2, dtype=dtype)
    w, b = normal(5, outputs, features, seed=3, dtype=dtype), normal(5, outputs, seed=4, dtype=dtype)
    inputs = [t.cuda().requires_grad_() for t in (x, w, b)]
    by = m.RowGroups(offsets.cuda())
    y = m.grouped_linear(inputs[0], inputs[1], by, inputs[2])
    grads = torch.autograd.grad(y, inputs, g.cuda())
    members = oracle.members(offsets, None, rows)
    check_grouped(x, w, b, g, members, y, grads)
    assert not y[:30].any() and not y[690:].any() and not grads[0][690:].any()
    # The same through an order, and of a few rows.
    order = torch.arange(rows, dtype=torch.int32).cuda()
    again = m.grouped_linear(inputs[0], inputs[1], m.RowGroups(by.offsets, order), inputs[2])
    assert torch.equal(again, y)
    few = m.RowGroups(torch.tensor([1, 3, 3, 3, 3, 9], dtype=torch.int32).cuda())
    got = m.grouped_linear(inputs[0][:10], inputs[1], few, inputs[2])
    want = oracle.grouped_linear(x[:10], w, oracle.members(few.offsets, None, 10), b)
    near(got, want, (features + 2) * E * oracle.grouped_linear(
        x[:10].abs(), w.abs(), oracle.members(few.offsets, None, 10), b.abs()), dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs,groups", [
    (310_001, 260, 260, 5), (150_000, 300, 40, 40), (60_001, 100, 130, 2000)])
def test_grouped_linear_of_many_rows_of_whole_numbers(dtype, rows, features, outputs, groups):
    """Every row counts: sums of small whole numbers stay below 2^24, which
    float32 holds exactly in any order, so each output is the exact sum,
    rounded once."""
    m = layers()
    gen = torch.Generator(device="cuda").manual_seed(7)

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=gen, device="cuda").to(dtype)

    x, g = whole(rows, features).requires_grad_(), whole(rows, outputs)
    w, b = whole(groups, outputs, features).requires_grad_(), whole(groups, outputs).requires_grad_()
    index = some_groups(rows, groups, 5, none=0.01).cuda()
    by = m.row_groups(index, groups)
    y = m.grouped_linear(x, w, by, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    bounds = by.offsets.tolist()
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for group in range(groups):
        at = by.order[bounds[group]:bounds[group + 1]].long()
        inside[at] = True
        part, d, matrix = x[at].detach().double(), g[at].double(), w[group].detach().double()
        assert torch.equal(y[at], (part @ matrix.t() + b[group].double()).to(dtype))
        assert torch.equal(dx[at], (d @ matrix).to(dtype))
        assert torch.equal(dw[group], (d.t() @ part).to(dtype))
        assert torch.equal(db[group], d.sum(0).to(dtype))
    assert not y[~inside].any() and not dx[~inside].any()


@gpu_test
def test_grouped_linear_gradients_asked_for_one_by_one():
    m = layers()
    index = some_groups(900, 6, 3)
    by, _ = grouped_by(index, 6)
    tensors = [normal(900, 40, seed=1), normal(6, 24, 40, seed=2), normal(6, 24, seed=3)]
    g = normal(900, 24, seed=4).cuda()
    for groups in (by, m.RowGroups(by.offsets)):
        every = [t.cuda().requires_grad_() for t in tensors]
        want = torch.autograd.grad(m.grouped_linear(every[0], every[1], groups, every[2]), every, g)
        for i in range(3):
            some = [t.cuda().requires_grad_(j == i) for j, t in enumerate(tensors)]
            y = m.grouped_linear(some[0], some[1], groups, some[2])
            (got,) = torch.autograd.grad(y, some[i], g)
            assert torch.equal(got, want[i])


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_keeps_bad_values_to_their_place(dtype):
    """A bad row shows in its own outputs and its own group's gradients; a
    bad row of no group nowhere."""
    m = layers()
    index = torch.arange(400) % 4 - 1
    by, _ = grouped_by(index, 3)
    x = normal(400, 64, seed=1, dtype=dtype)
    w, g = normal(3, 32, 64, seed=2, dtype=dtype), normal(400, 32, seed=3, dtype=dtype)
    outs = []
    for bad in (False, True):
        held, grad = x.clone(), g.clone()
        if bad:
            held[4], held[8, 3], grad[4] = math.nan, math.inf, math.inf  # rows of no group
            held[5] = math.nan                                          # of group 0
        inputs = [t.cuda().requires_grad_() for t in (held, w)]
        y = m.grouped_linear(*inputs, by)
        outs.append((y, *torch.autograd.grad(y, inputs, grad.cuda())))
    (y0, dx0, dw0), (y1, dx1, dw1) = outs
    rows = torch.arange(400, device="cuda") != 5
    assert torch.equal(y0[rows], y1[rows]) and y1[5].isnan().all()
    assert torch.equal(dx0, dx1) and torch.equal(dw0[1:], dw1[1:]) and dw1[0].isnan().all()


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_shapes_and_strides(dtype):
    m = layers()
    base = normal(30, 4, 200, seed=1, dtype=dtype).cuda()
    w = normal(3, 96, 80, seed=2, dtype=dtype).cuda()
    for view in (lambda t: t[:, 1, :96], lambda t: t[:, 2, 3:99], lambda t: t[:, :3, 8:104],
                 lambda t: t.transpose(0, 2)[:96].transpose(0, 1).transpose(1, 2)[..., :96],
                 lambda t: t[:1, 0, :96].expand(60, 96)):
        x = view(base)
        if x.shape[-1] != 96:
            continue
        rows = x.numel() // 96
        by = m.row_groups((torch.arange(rows) % 4 - 1).cuda(), 3)
        for matrix in (w.transpose(1, 2), w.transpose(1, 2).contiguous()):  # [3, 80, 96]
            got, want = [], []
            for source, out in ((x, got), (x.contiguous(), want)):
                on = source.detach().requires_grad_()
                weight = matrix.detach().requires_grad_()
                y = m.grouped_linear(on, weight, by)
                out += [y, *torch.autograd.grad(y, (on, weight),
                                                torch.ones(1, dtype=dtype, device="cuda").expand_as(y))]
            assert got[0].shape == (*x.shape[:-1], 80)
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@gpu_test
def test_grouped_linear_of_no_rows():
    m = layers()
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w = torch.ones(3, 4, 8, device="cuda", requires_grad=True)
    b = torch.ones(3, 4, device="cuda", requires_grad=True)
    y = m.grouped_linear(x, w, m.row_groups(torch.zeros(0, dtype=torch.int64, device="cuda"), 3), b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 4) and dx.shape == (0, 8) and not dw.any() and not db.any()


@gpu_test
def test_grouped_linear_refusals():
    m = layers()
    x, w = torch.zeros(6, 8, device="cuda"), torch.zeros(3, 4, 8, device="cuda")
    by = m.row_groups(torch.zeros(6, dtype=torch.int32, device="cuda"), 3)
    with pytest.raises(TypeError, match="RowGroups"):
        m.grouped_linear(x, w, by.offsets)
    for weight in (w[0], w[..., :7], torch.zeros(0, 4, 8, device="cuda")):
        with pytest.raises(ValueError, match="weight must have shape"):
            m.grouped_linear(x, weight, by)
    with pytest.raises(ValueError, match="type of x"):
        m.grouped_linear(x, w.half(), by)
    with pytest.raises(ValueError, match="bias must have shape"):
        m.grouped_linear(x, w, by, torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError, match="of 3 groups, not 2"):
        m.grouped_linear(x, w[:2], by)
    with pytest.raises(ValueError, match="order of 6 rows, x has 5"):
        m.grouped_linear(x[:5], w, by)
    with pytest.raises(ValueError, match="groups must be on the device"):
        m.grouped_linear(x, w, m.RowGroups(by.offsets.cpu(), by.order.cpu()))
    y = m.grouped_linear(x.requires_grad_(), w, by)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="grouped_linear is differentiable once"):
        dx.sum().backward()


# --------------------------------------------------------------------------
# GPU: linear layers with adapters by group

# An inner row of a 2-byte type is kept in two parts: to 2^-16 of its value in
# bfloat16, whose first part is cut off, and in float16 to 2^-21 of its row's
# largest (its second part may be below the type's normal range).
INNER = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -21}


def near_or_past(got, expected, error, dtype):
    """near, but for what is past the type's largest: an infinity by the rounding
    itself (float16: from 65520 on)."""
    most = torch.finfo(dtype).max
    past = expected.abs() - error > most * (1 + torch.finfo(dtype).eps / 2)
    got = got.detach().cpu().double()
    assert torch.equal(got[past], torch.sign(expected[past]) * math.inf)
    edge = ~past & (expected.abs() + error >= most)
    assert edge.sum() <= 1 + edge.numel() // 1000
    fine = ~past & ~edge
    near(got[fine], expected[fine], error[fine], dtype)


def check_adapted(x, w, b, a, u, g, scale, members, y, grads):
    """Errors: sums of float32, the inner rows' parts, and their own sums' errors
    on the way through the other products."""
    dtype, rank = x.dtype, a.shape[1]
    rows, features, outputs = len(x), x.shape[1], w.shape[0]
    want = oracle.adapted_linear(x, w, a, u, members, b, scale, g)
    low, high = w.abs(), None if b is None else b.abs()
    size = oracle.adapted_linear(x.abs(), low, a.abs(), u.abs(), members, high, abs(scale), g.abs())
    terms = features + outputs + rank + 8

    def inner_error(sum_error):
        return sum_error * E + INNER[dtype]

    inner = torch.zeros(rows, rank, dtype=torch.float64)
    back = torch.zeros(rows, rank, dtype=torch.float64)
    for group, at in enumerate(members):
        inner[at] = abs(scale) * (x[at].double().abs() @ a[group].double().abs().t())
        back[at] = abs(scale) * (g[at].double().abs() @ u[group].double().abs())
    # float16's parts go by the row's largest.
    if dtype == torch.float16:
        inner, back = (t.amax(1, keepdim=True).expand_as(t) for t in (inner, back))
    narrow = [torch.zeros(rows, outputs, dtype=torch.float64), torch.zeros(rows, features,
                                                                         dtype=torch.float64),
              torch.zeros_like(a, dtype=torch.float64), torch.zeros_like(u, dtype=torch.float64)]
    for group, at in enumerate(members):
        narrow[0][at] = inner[at] @ u[group].double().abs().t()
        narrow[1][at] = back[at] @ a[group].double().abs()
        narrow[2][group] = back[at].t() @ x[at].double().abs()
        narrow[3][group] = g[at].double().abs().t() @ inner[at]
    most = max([len(m) for m in members] + [1]) + 2
    near_or_past(y.reshape(rows, outputs), want[0],
         terms * E * size[0] + inner_error(features + 2) * narrow[0], dtype)
    near_or_past(grads[0].reshape(rows, features), want[1],
         terms * E * size[1] + inner_error(outputs + 2) * narrow[1], dtype)
    near_or_past(grads[1], want[2], most * E * size[2] + inner_error(outputs + 2) * narrow[2], dtype)
    near_or_past(grads[2], want[3], most * E * size[3] + inner_error(features + 2) * narrow[3], dtype)


def adapted_case(rows, features, outputs, groups, rank, dtype, bias=True, seed=31, scale=0.7,
                 index=None, by=None, size=1.0):
    m = layers()
    x = normal(rows, features, seed=seed, dtype=dtype)
    w = normal(outputs, features, seed=seed + 1, dtype=dtype, scale=features ** -0.5)
    b = normal(outputs, seed=seed + 2, dtype=dtype) if bias else None
    a = normal(groups, rank, features, seed=seed + 3, dtype=dtype, scale=size * features ** -0.5)
    u = normal(groups, outputs, rank, seed=seed + 4, dtype=dtype, scale=rank ** -0.5)
    g = normal(rows, outputs, seed=seed + 5, dtype=dtype)
    if by is None:
        index = some_groups(rows, groups, seed) if index is None else index
        by, members = grouped_by(index, groups)
    else:
        members = oracle.members(by.offsets, by.order, rows)
    on, wc, ac, uc = (t.cuda().requires_grad_(i != 1) for i, t in enumerate((x, w, a, u)))
    bc = None if b is None else b.cuda()
    y = m.adapted_linear(on, wc, ac, uc, by, bc, scale)
    grads = torch.autograd.grad(y, (on, ac, uc), g.cuda())
    with torch.no_grad():
        assert torch.equal(m.adapted_linear(on, wc, ac, uc, by, bc, scale), y)
    check_adapted(x, w, b, a, u, g, scale, members, y, grads)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs,groups,rank", [
    (1, 1, 1, 1, 1), (1, 1024, 57, 8, 16), (4, 64, 64, 8, 5), (16, 33, 18, 3, 64), (17, 8, 8, 5, 4),
    (40, 5, 3, 2, 2), (64, 96, 57, 64, 16), (127, 130, 63, 4, 33), (300, 187, 18, 7, 5),
    (1000, 40, 72, 300, 8), (2500, 264, 136, 6, 32), (1024, 64, 57, 16, 17), (5000, 128, 128, 12, 64),
    (200, 1100, 40, 3, 16), (200, 40, 1100, 3, 16), (90, 1030, 1030, 2, 48), (700, 512, 512, 5, 16),
    (900, 256, 256, 3, 31)])
def test_adapted_linear(dtype, rows, features, outputs, groups, rank):
    adapted_case(rows, features, outputs, groups, rank, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("features,outputs,rank", [
    (64, 256, 16), (128, 512, 16), (190, 256, 40), (256, 256, 16), (256, 256, 33), (320, 200, 8),
    (512, 512, 16), (512, 512, 40)])
def test_adapted_linear_of_wide_panels(dtype, features, outputs, rank):
    """Rows enough for the widest panels, steps that the adapters' chunks make a
    whole number of those under way and others, and matrices that leave no room in
    LDS for the adapters beside the widest."""
    adapted_case(3000, features, outputs, 5, rank, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("features,outputs", [(64, 256), (190, 512), (512, 512), (256, 300)])
def test_grouped_linear_of_wide_panels(dtype, features, outputs):
    grouped_case(3000, features, outputs, 5, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_adapted_linear_of_special_groups(dtype):
    m = layers()
    adapted_case(500, 64, 40, 5, 8, dtype, bias=False, scale=-2.0)
    none = torch.full((200,), -1)
    adapted_case(200, 64, 40, 5, 8, dtype, index=none)           # no row has an adapter
    adapted_case(200, 64, 40, 5, 8, dtype, index=none + 4)       # one has all
    adapted_case(3000, 64, 40, 5, 8, dtype, index=torch.arange(3000) % 5)
    adapted_case(130, 64, 40, 130, 8, dtype, index=torch.arange(130))  # a row each
    adapted_case(2000, 24, 8, 3000, 3, dtype)
    adapted_case(300, 64, 40, 5, 8, dtype, scale=0.0)
    offsets = torch.tensor([30, 30, 200, 455, 455, 690], dtype=torch.int32).cuda()
    adapted_case(700, 64, 40, 5, 8, dtype, by=m.RowGroups(offsets))
    adapted_case(10, 64, 40, 2, 8, dtype, by=m.RowGroups(
        torch.tensor([1, 3, 8], dtype=torch.int32).cuda()))


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 12])
def test_adapted_linear_of_small_and_large_inner_rows(dtype, size):
    """Inner values far from 1, past float16's largest where `size` is 2^12:
    their own range is float32's. Some of down's gradients are past it where
    `size` is 2^-12 (scale 2^12)."""
    adapted_case(400, 64, 40, 5, 8, dtype, size=size, scale=1 / size)
    adapted_case(400, 64, 40, 5, 8, dtype, size=size, scale=32 / size ** 2)
    adapted_case(9, 64, 40, 5, 8, dtype, size=size, scale=1 / size)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_adapted_linear_gradients_asked_for_one_by_one(dtype):
    """The shared layer's are linear's."""
    m = layers()
    index = some_groups(900, 6, 3)
    by, _ = grouped_by(index, 6)
    tensors = [normal(900, 40, seed=1, dtype=dtype), normal(24, 40, seed=2, dtype=dtype),
               normal(6, 8, 40, seed=3, dtype=dtype), normal(6, 24, 8, seed=4, dtype=dtype),
               normal(24, seed=5, dtype=dtype)]
    g = normal(900, 24, seed=6, dtype=dtype).cuda()
    for groups in (by, m.RowGroups(by.offsets)):
        every = [t.cuda().requires_grad_() for t in tensors]
        want = torch.autograd.grad(m.adapted_linear(*every[:4], groups, every[4]), every, g)
        plain = torch.autograd.grad(m.linear(every[0], every[1], every[4]), (every[1], every[4]), g)
        assert torch.equal(want[1], plain[0]) and torch.equal(want[4], plain[1])
        for i in range(5):
            some = [t.cuda().requires_grad_(j == i) for j, t in enumerate(tensors)]
            y = m.adapted_linear(*some[:4], groups, some[4])
            (got,) = torch.autograd.grad(y, some[i], g)
            assert torch.equal(got, want[i])


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_adapted_linear_keeps_bad_values_to_their_place(dtype):
    m = layers()
    index = torch.arange(400) % 4 - 1
    by, _ = grouped_by(index, 3)
    x, w = normal(400, 64, seed=1, dtype=dtype), normal(32, 64, seed=2, dtype=dtype)
    a, u = normal(3, 8, 64, seed=3, dtype=dtype), normal(3, 32, 8, seed=4, dtype=dtype)
    g = normal(400, 32, seed=5, dtype=dtype)
    outs = []
    for bad in (False, True):
        held, grad = x.clone(), g.clone()
        if bad:
            held[4], grad[4] = math.nan, math.inf  # a row of no group
            held[5] = math.nan                     # of group 0
        on, ac, uc = (t.cuda().requires_grad_() for t in (held, a, u))
        y = m.adapted_linear(on, w.cuda(), ac, uc, by)
        outs.append((y, *torch.autograd.grad(y, (on, ac, uc), grad.cuda())))
    (y0, dx0, da0, du0), (y1, dx1, da1, du1) = outs
    rows = torch.ones(400, dtype=torch.bool, device="cuda")
    rows[4:6] = False
    assert torch.equal(y0[rows], y1[rows]) and y1[4:6].isnan().all()
    assert torch.equal(dx0[rows], dx1[rows])
    assert torch.equal(da0[1:], da1[1:]) and da1[0].isnan().all()
    assert torch.equal(du0[1:], du1[1:]) and du1[0].isnan().all()


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [9, 600])
def test_adapted_linear_shapes_and_strides(dtype, rows):
    m = layers()
    base = normal(rows, 4, 200, seed=1, dtype=dtype).cuda()
    w = normal(40, 96, seed=2, dtype=dtype).cuda()
    a, u = normal(3, 8, 96, seed=3, dtype=dtype).cuda(), normal(3, 40, 8, seed=4, dtype=dtype).cuda()
    for view in (lambda t: t[:, 1, :96], lambda t: t[:, 2, 3:99], lambda t: t[:, :3, 8:104],
                 lambda t: t[:1, 0, :96].expand(rows, 96)):
        x = view(base)
        by = m.row_groups((torch.arange(x.numel() // 96) % 4 - 1).cuda(), 3)
        outs = []
        for source, turned in ((x, False), (x.contiguous(), True)):
            on, down, up = (t.detach().requires_grad_() for t in (
                source, a.transpose(1, 2).contiguous().transpose(1, 2) if turned else a, u))
            y = m.adapted_linear(on, w.t().contiguous().t() if turned else w, down, up, by)
            outs.append((y, *torch.autograd.grad(
                y, (on, down, up), torch.ones(1, dtype=dtype, device="cuda").expand_as(y))))
        assert outs[0][0].shape == (*x.shape[:-1], 40)
        for got, want in zip(*outs):
            assert torch.equal(got, want)


@gpu_test
def test_adapted_linear_of_no_rows():
    m = layers()
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w, b = torch.ones(4, 8, device="cuda", requires_grad=True), torch.ones(4, device="cuda")
    a = torch.ones(3, 2, 8, device="cuda", requires_grad=True)
    u = torch.ones(3, 4, 2, device="cuda", requires_grad=True)
    by = m.row_groups(torch.zeros(0, dtype=torch.int64, device="cuda"), 3)
    y = m.adapted_linear(x, w, a, u, by, b)
    grads = torch.autograd.grad(y.sum(), (x, w, a, u))
    assert y.shape == (0, 4) and not any(t.any() for t in grads)


@gpu_test
def test_adapted_linear_refusals():
    m = layers()
    x, w = torch.zeros(6, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    a, u = torch.zeros(3, 2, 8, device="cuda"), torch.zeros(3, 4, 2, device="cuda")
    by = m.row_groups(torch.zeros(6, dtype=torch.int32, device="cuda"), 3)
    with pytest.raises(TypeError, match="RowGroups"):
        m.adapted_linear(x, w, a, u, None)
    with pytest.raises(TypeError, match="down must be"):
        m.adapted_linear(x, w, None, u, by)
    for down in (a[0], a[..., :7], torch.zeros(3, 65, 8, device="cuda")):
        with pytest.raises(ValueError, match="down must have shape"):
            m.adapted_linear(x, w, down, u, by)
    for up in (u[:2], u.transpose(1, 2)):
        with pytest.raises(ValueError, match="up must have shape"):
            m.adapted_linear(x, w, a, up, by)
    with pytest.raises(ValueError, match="type of x"):
        m.adapted_linear(x, w, a.half(), u, by)
    with pytest.raises(ValueError, match="weight must have shape"):
        m.adapted_linear(x, w[:, :7], a, u, by)
    with pytest.raises(ValueError, match="of 3 groups, not 2"):
        m.adapted_linear(x, w, a[:2], u[:2], by)
    for scale in (math.inf, math.nan, 1e39):
        with pytest.raises(ValueError, match="scale must be finite"):
            m.adapted_linear(x, w, a, u, by, scale=scale)
    with pytest.raises(ValueError, match="scale has no gradient"):
        m.adapted_linear(x, w, a, u, by, scale=torch.ones((), requires_grad=True))
    y = m.adapted_linear(x.requires_grad_(), w, a, u, by)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="adapted_linear is differentiable once"):
        dx.sum().backward()


# --------------------------------------------------------------------------
# GPU: all of them


def parts_step(dtype=torch.bfloat16, rows=700, seed=51, offsets_only=False):
    """Leaves and a function that runs the operators as a decoder in parts does:
    a layer by part, dropout, a shared layer with the parts' adapters."""
    m = layers()
    x = normal(rows, 72, seed=seed, dtype=dtype)
    w, b = normal(6, 64, 72, seed=seed + 1, dtype=dtype, scale=0.1), normal(6, 64, seed=seed + 2,
                                                                          dtype=dtype)
    shared = normal(57, 64, seed=seed + 3, dtype=dtype, scale=0.1)
    bias = normal(57, seed=seed + 4, dtype=dtype)
    down = normal(6, 8, 64, seed=seed + 5, dtype=dtype, scale=0.1)
    up = normal(6, 57, 8, seed=seed + 6, dtype=dtype, scale=0.3)
    index = some_groups(rows, 6, seed)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, shared, bias, down, up)]
    on_device = index.cuda()
    grad = normal(rows, 57, seed=seed + 7, dtype=dtype).cuda()

    def run(keep=None):
        x, w, b, shared, bias, down, up = leaves
        by = m.row_groups(on_device, 6)
        h = m.grouped_linear(x, w, by, b)
        d = m.dropout(h, 0.25, 99)
        y = m.adapted_linear(d, shared, down, up, by, bias, scale=0.5)
        if keep is not None:
            keep.update(by=by, h=h, d=d)
            h.retain_grad()
            d.retain_grad()
        return y

    return leaves, grad, run


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_operators_together(dtype):
    """Each operator against its formula at what the one before gave it, forward
    and backward."""
    m = layers()
    leaves, grad, run = parts_step(dtype)
    kept = {}
    y = run(kept)
    y.backward(grad)
    x, w, b, shared, bias, down, up = (t.detach().cpu() for t in leaves)
    h, d = kept["h"].detach().cpu(), kept["d"].detach().cpu()
    members = oracle.members(kept["by"].offsets, kept["by"].order, len(x))
    check_grouped(x, w, b, kept["h"].grad.cpu(), members, kept["h"],
                  [leaves[0].grad, leaves[1].grad, leaves[2].grad])
    check_dropout(h, kept["d"].grad.cpu(), 0.25, 99, kept["d"], kept["h"].grad)
    check_adapted(d, shared, bias, down, up, grad.cpu(), 0.5, members, y,
                  [kept["d"].grad, leaves[5].grad, leaves[6].grad])
    plain = torch.autograd.grad(m.linear(kept["d"].detach(), leaves[3], leaves[4]), leaves[3:5],
                                grad)
    assert torch.equal(leaves[3].grad, plain[0]) and torch.equal(leaves[4].grad, plain[1])


@gpu_test
def test_results_repeat_bit_for_bit_on_any_stream():
    leaves, grad, run = parts_step()
    want = None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            y = run()
            got = (y, *torch.autograd.grad(y, leaves, grad))
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu_test
def test_operators_in_graphs():
    """Two graphs of the forward and backward passes, replayed in turn with
    eager work between, over inputs and groups that change."""
    steps = [parts_step(rows=700), parts_step(torch.float32, rows=9000, seed=81)]
    graphs, outs = [], []
    for leaves, grad, run in steps:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(run(), leaves, grad)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = run()
            out = (y.detach(), *torch.autograd.grad(y, leaves, grad))
        del y
        graphs.append(graph)
        outs.append(out)
    for round_ in range(3):
        for (leaves, grad, run), graph, out in zip(steps, graphs, outs):
            with torch.no_grad():
                for t in leaves:
                    t.mul_(1 + 0.25 * round_)
            graph.replay()
            torch.cuda.synchronize()
            y = run()
            want = (y, *torch.autograd.grad(y, leaves, grad))
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            del y, want


@gpu_test
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_against_differences(dtype):
    """The operators are linear in each of their inputs, and small whole numbers
    leave nothing to round: differences give the gradients exactly."""
    m = layers()
    gen = torch.Generator().manual_seed(3)

    def whole(*shape, most=1):
        return torch.randint(-most, most + 1, shape, generator=gen).to(dtype).cuda()

    by, _ = grouped_by(some_groups(40, 3, 4), 3)
    cases = [(lambda *t: m.grouped_linear(t[0], t[1], by, t[2]),
              [whole(40, 12), whole(3, 9, 12), whole(3, 9)], whole(40, 9)),
             (lambda *t: m.adapted_linear(t[0], w, t[1], t[2], by, scale=2.0),
              [whole(40, 12), whole(3, 2, 12), whole(3, 9, 2)], whole(40, 9))]
    w = whole(9, 12)
    for call, inputs, g in cases:
        for t in inputs:
            t.requires_grad_()
        grads = torch.autograd.grad(call(*inputs), inputs, g)
        for i, grad in enumerate(grads):
            step = whole(*inputs[i].shape)
            with torch.no_grad():
                moved = [[t + sign * step if j == i else t for j, t in enumerate(inputs)]
                         for sign in (1, -1)]
                up, down = ((call(*at).double() * g.double()).sum() for at in moved)
            assert (up - down) / 2 == (grad.double() * step.double()).sum()


@gpu_test
def test_offsets_past_32_bits():
    """Rows that lie over 2^32 values apart, and results of more values."""
    m = layers()
    rows, stride = 70_000, 65_536
    base = torch.empty(rows, stride, dtype=torch.float16, device="cuda")  # 9.2 GB
    x = base[:, 100:140]
    x.copy_(normal(rows, 40, seed=1, dtype=torch.float16))
    dense = x.contiguous()
    by = m.row_groups((torch.arange(rows) % 5 - 1).cuda(), 4)
    w, b = normal(4, 24, 40, seed=2, dtype=torch.float16).cuda(), None
    a, u = (normal(4, 8, 40, seed=3, dtype=torch.float16).cuda(),
            normal(4, 24, 8, seed=4, dtype=torch.float16).cuda())
    g = normal(rows, 24, seed=5, dtype=torch.float16).cuda()
    outs = []
    for source in (x, dense):
        t, wt, at, ut = (v.detach().requires_grad_() for v in (source, w, a, u))
        y = m.grouped_linear(t, wt, by, b)
        z = m.adapted_linear(t, w[0], at, ut, by)
        outs.append((y, z, *torch.autograd.grad(y, (t, wt), g), *torch.autograd.grad(z, (t, at, ut), g),
                     m.dropout(source, 0.5, 3)))
    assert all(torch.equal(p, q) for p, q in zip(*outs))
    del outs, base, x, y, z
    rows = 4_300_000
    x = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 4_194_303, 4_194_304, rows - 1], device="cuda")
    x[at] = 1
    w = torch.ones(2, 1024, 8, dtype=torch.bfloat16, device="cuda")
    w[1] = 2
    index = torch.zeros(rows, dtype=torch.int32, device="cuda")
    index[at[2:]] = 1
    y = m.grouped_linear(x, w, m.row_groups(index, 2))  # 4.4e9 values
    want = torch.tensor([8.0, 8, 16, 16, 16], device="cuda", dtype=torch.bfloat16)
    assert torch.equal(y[at], want[:, None].expand(5, 1024)) and int(y[:, 5].count_nonzero()) == 5
    kept = m.dropout(y[at[2:4]], 0.5, 3)
    whole = m.dropout(y, 0.5, 3)
    some = oracle.dropout(y[at].cpu().float(), 0.5, 3, rows=at.tolist())
    assert torch.equal(whole[at].cpu().double(), some) and kept.shape == (2, 1024)


@gpu_test
def test_wrong_groups_stay_inside():
    """Offsets that fall or pass the rows, and rows that are not there: results
    are not defined, but every access is held to what exists, and later calls are
    right."""
    m = layers()
    leaves, grad, run = parts_step()
    want = run()
    x, w, b, shared, bias, down, up = leaves
    rows = len(x)
    for offsets, order in (([0, 300, 100, 50, 600, 650, 700], None),
                           ([-5, 10, 2_000_000, 20, 30, 1 << 30, 700], None),
                           ([700] * 7, None), ([0] * 7, None),
                           ([0, 100, 200, 300, 400, 500, 700], [-1, 1 << 30, 5, 5] * 175)):
        by = m.RowGroups(torch.tensor(offsets, dtype=torch.int32).cuda(),
                         None if order is None else torch.tensor(order, dtype=torch.int32).cuda())
        for few in (rows, 12):
            groups = by if order is None or few == rows else m.RowGroups(by.offsets,
                                                                       by.order[:few].contiguous())
            for y in (m.grouped_linear(x[:few], w, groups, b),
                      m.adapted_linear(leaves[0][:few, :64], shared, down, up, groups, bias)):
                torch.autograd.grad(y.sum(), leaves, allow_unused=True)
    torch.cuda.synchronize()
    assert torch.equal(run(), want)


@gpu_test
def test_lazily_negated_views():
    m = layers()
    z = torch.complex(normal(50, 24, seed=1), normal(50, 24, seed=2)).cuda()
    view = z.conj().imag
    assert view.is_neg()
    by = m.row_groups((torch.arange(50) % 3).cuda(), 3)
    w, a, u = (normal(3, 16, 24, seed=3).cuda(), normal(3, 4, 24, seed=4).cuda(),
               normal(3, 16, 4, seed=5).cuda())
    plain = view.resolve_neg()
    assert torch.equal(m.grouped_linear(view, w, by), m.grouped_linear(plain, w, by))
    assert torch.equal(m.adapted_linear(view, w[0], a, u, by), m.adapted_linear(plain, w[0], a, u, by))
    assert torch.equal(m.dropout(view, 0.5, 1), m.dropout(plain, 0.5, 1))


@gpu_test
def test_groups_may_not_change_before_the_backward_pass():
    m = layers()
    x = normal(30, 8, seed=1).cuda().requires_grad_()
    w = normal(2, 4, 8, seed=2).cuda()
    a, u = normal(2, 3, 8, seed=3).cuda(), normal(2, 4, 3, seed=4).cuda()
    for call in (lambda by: m.grouped_linear(x, w, by),
                 lambda by: m.adapted_linear(x, w[0], a, u, by)):
        for change in ("offsets", "order"):
            by = m.row_groups((torch.arange(30) % 2).cuda(), 2)
            y = call(by)
            getattr(by, change).add_(0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()


def parts_calls(device="cpu"):
    m = layers()
    w, a = torch.ones(2, 4, 8, device=device), torch.ones(2, 3, 8, device=device)
    u, shared = torch.ones(2, 4, 3, device=device), torch.ones(4, 8, device=device)
    by = m.RowGroups(torch.tensor([0, 1, 2], dtype=torch.int32, device=device))
    return {"dropout": lambda t: m.dropout(t, 0.5, 1),
            "grouped_linear": lambda t: m.grouped_linear(t, w, by),
            "adapted_linear": lambda t: m.adapted_linear(t, shared, a, u, by)}


def test_forward_mode_and_tracing_are_refused():
    from test_layers import refuses_what_would_lose_a_result
    from torch.fx.experimental.proxy_tensor import make_fx

    m = layers()
    refuses_what_would_lose_a_result(parts_calls(), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="row_groups cannot be traced"):
        make_fx(lambda t: m.row_groups(t, 2).order)(torch.zeros(4, dtype=torch.int32))


@gpu_test
def test_forward_mode_and_tracing_are_refused_on_the_device():
    from test_layers import refuses_what_would_lose_a_result

    refuses_what_would_lose_a_result(parts_calls("cuda"), torch.ones(2, 8, device="cuda"))


@gpu_test
def test_second_derivatives_are_refused():
    m = layers()
    x = normal(4, 32, seed=1).cuda().requires_grad_()
    (dx,) = torch.autograd.grad(m.dropout(x, 0.5, 1).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="dropout is differentiable once"):
        dx.sum().backward()


def test_c_entry_points_of_layers_by_group_refuse_bad_arguments():
    from diff_gabor_splatting_amd import _native

    lib, p = _native.lib, ctypes.c_void_p(256)
    forward = lambda *t: lib.gs_grouped_linear_forward(*t, None)  # noqa: E731
    refused(lib, forward(3, p, 8, p, p, p, p, 4, 2, 8, 8, p), 1, "unknown type")
    refused(lib, forward(0, p, 7, p, p, p, p, 4, 2, 8, 8, p), 1, "overlap")
    refused(lib, forward(0, p, 8, p, p, p, None, 4, 2, 8, 8, p), 1, "null")
    refused(lib, forward(0, p, 8, None, p, p, p, 4, 2, 8, 8, p), 1, "null")
    refused(lib, forward(0, p, 8, p, p, p, p, 1 << 31, 2, 8, 8, p), 2, "rows")
    refused(lib, forward(0, p, 8, p, p, p, p, 4, 0, 8, 8, p), 1, "groups")
    refused(lib, forward(0, p, 8, p, p, p, p, 4, (1 << 20) + 1, 8, 8, p), 1, "groups")
    refused(lib, forward(0, p, 8, p, p, p, p, 4, 2, 8, 1 << 20, p), 1, "at most")
    assert forward(0, None, 8, None, None, None, None, 0, 2, 8, 8, None) == 0
    refused(lib, lib.gs_grouped_linear_backward_input(0, p, 8, p, p, p, 4, 2, 8, 8, None, None), 1,
            "null")
    need = lib.gs_grouped_linear_backward_weight_workspace_size(0, 5000, 4, 64, 64)
    assert need > 0
    refused(lib, lib.gs_grouped_linear_backward_weight(0, p, 64, p, 64, p, p, 5000, 4, 64, 64, p, p,
                                                       p, need - 1, None), 4, "workspace")
    refused(lib, lib.gs_grouped_linear_backward_weight(0, p, 64, None, 64, p, p, 5000, 4, 64, 64, p,
                                                       p, p, need, None), 1, "null")
    size = lib.gs_adapted_linear_inner_size(100, 16)
    assert size >= 100 * 16 * 4

    def adapted(dtype=0, scale=1.0, rank=16, bytes=size, inner=p, up=p):
        return lib.gs_adapted_linear_forward(dtype, p, 8, p, p, p, up, scale, p, p, 100, 2, 8, 8,
                                             rank, inner, bytes, p, None)

    refused(lib, adapted(dtype=7), 1, "unknown type")
    refused(lib, adapted(scale=math.inf), 1, "scale")
    refused(lib, adapted(rank=65), 1, "rank")
    refused(lib, adapted(rank=0), 1, "rank")
    refused(lib, adapted(bytes=size - 1), 4, "inner rows")
    refused(lib, adapted(inner=None), 4, "inner rows")
    refused(lib, adapted(up=None), 1, "null")
    refused(lib, lib.gs_adapted_linear_backward_input(0, p, 8, None, p, p, 1.0, p, p, 100, 2, 8, 8,
                                                      16, p, size, p, None), 1, "null")
    need = lib.gs_adapted_linear_backward_adapters_workspace_size(5000, 2, 64, 64, 16)
    assert need > 0
    refused(lib, lib.gs_adapted_linear_backward_adapters(0, p, 64, p, 64, p, p, p, p, 5000, 2, 64,
                                                         64, 16, p, p, p, need - 1, None), 4,
            "workspace")
    refused(lib, lib.gs_adapted_linear_backward_adapters(0, p, 64, p, 64, None, p, p, p, 5000, 2, 64,
                                                         64, 16, p, p, p, need, None), 1, "null")


def test_python_layers_by_group_refuse_cpu_tensors():
    for call in parts_calls().values():
        with pytest.raises(ValueError, match="on a HIP device"):
            call(torch.zeros(2, 8))
