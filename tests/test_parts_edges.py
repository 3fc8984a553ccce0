"""Layers by group at their edges: infinities, scales far from one, gradients
asked for alone, the widest tiles and the joins of many parts, groups that
change under a captured graph, and memory beside the results.

Tolerances as in test_parts.py.
"""

import ctypes
import math

import pytest
import torch

from oracle import parts as oracle
from test_layers import DTYPES, E, gpu_test, layers, near, normal
from test_parts import INNER, adapted_case, grouped_by, some_groups

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

# --------------------------------------------------------------------------
# Scales far from one


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [2.0 ** -90, 2.0 ** 90, -(2.0 ** 100)])
def test_adapted_linear_of_scales_far_from_one(dtype, scale):
    """Inner values in float32's range, whatever the type: float16's results
    are infinities there, and no NaN."""
    adapted_case(400, 64, 40, 5, 8, dtype, scale=scale)
    adapted_case(9, 64, 40, 5, 8, dtype, scale=scale)


@gpu_test
@pytest.mark.parametrize("scale", [2.0 ** 90, -(2.0 ** 100)])
def test_wide_float16_layers_of_large_scales(scale):
    """Sums of 1100 terms by tiles. Where the formula's value is past float16's
    largest by more than the sums' error, it is an infinity of its sign. The
    error is (1100 + 2) e of what the magnitudes add up to, 8 (the rank) * 21
    (1100 products of mean 0.64 / sqrt(1100)) * 0.28 (of `up`) = 48 times the
    scale, and as much again of the shared terms' bound: 6e-3 of values whose
    spread is about 1, so half a percent of them say nothing."""
    m, dtype = layers(), torch.float16
    rows, features, outputs, groups, rank = 60, 1100, 40, 3, 8
    x, g = normal(rows, features, seed=31, dtype=dtype), normal(rows, outputs, seed=36, dtype=dtype)
    w = normal(outputs, features, seed=32, dtype=dtype, scale=features ** -0.5)
    a = normal(groups, rank, features, seed=34, dtype=dtype, scale=features ** -0.5)
    u = normal(groups, outputs, rank, seed=35, dtype=dtype, scale=rank ** -0.5)
    by, members = grouped_by(some_groups(rows, groups, 31), groups)
    on = x.cuda().requires_grad_()
    y = m.adapted_linear(on, w.cuda(), a.cuda(), u.cuda(), by, scale=scale)
    (dx,) = torch.autograd.grad(y, on, g.cuda())
    want = oracle.adapted_linear(x, w, a, u, members, None, scale, g)
    size = oracle.adapted_linear(x.abs(), w.abs(), a.abs(), u.abs(), members, None, abs(scale),
                                 g.abs())
    inside = torch.cat(members)
    for got, expected, total in zip((y, dx), want, size):
        got, error = got.detach().cpu().double(), 2 * (features + outputs) * E * total
        assert not got.isnan().any()
        past = expected.abs() - error > 65520
        assert torch.equal(got[past], torch.sign(expected[past]) * math.inf)
        assert past[inside].double().mean() > 0.97
        none = torch.ones(rows, dtype=torch.bool)
        none[inside] = False
        near(got[none], expected[none], error[none], dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", [(9, 64), (400, 64), (60, 1100)])
def test_adapted_linear_of_large_inner_rows_that_meet_zeros(dtype, rows, features):
    """Adapters whose `up` is still zero, as training begins: the shared layer's
    values, whatever the inner rows are."""
    m = layers()
    by, _ = grouped_by(some_groups(rows, 3, 4), 3)
    x, w = normal(rows, features, seed=1, dtype=dtype).cuda(), normal(40, features, seed=2,
                                                                   dtype=dtype).cuda()
    a = normal(3, 8, features, seed=3, dtype=dtype).cuda()
    u = torch.zeros(3, 40, 8, dtype=dtype, device="cuda")
    want = m.adapted_linear(x, w, a, u, by, scale=0.0)
    for scale in (1.0, 2.0 ** 20, 2.0 ** 60, 2.0 ** 80, 2.0 ** 110):
        assert torch.equal(m.adapted_linear(x, w, a, u, by, scale=scale), want), scale


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [9, 300])
def test_inner_rows_hold_17_bits(dtype, rows):
    """131071 is 17 ones: y is what is left of it beside 131072, forward and
    backward."""
    m = layers()
    by, _ = grouped_by(torch.zeros(rows, dtype=torch.int64), 1)
    x = torch.zeros(rows, 64, dtype=dtype)
    x[:, :2] = torch.tensor([1.0, -1.0])
    a = torch.zeros(1, 2, 64, dtype=dtype)
    a[0, 0, 0], a[0, 0, 1], a[0, 1, 0] = 512, 2.0 ** -8, 512  # 512 - 2^-8 and 512
    u = torch.zeros(1, 40, 2, dtype=dtype)
    u[0, :, 0], u[0, :, 1] = 1, -1
    on, w = x.cuda().requires_grad_(), torch.zeros(40, 64, dtype=dtype, device="cuda")
    y = m.adapted_linear(on, w, a.cuda(), u.cuda(), by, scale=256.0)
    assert (y == -1).all()
    # The gradient's inner row: 131071 for rank 0 and 131072 for rank 1.
    u = torch.zeros(1, 40, 2, dtype=dtype)
    u[0, 0, 0], u[0, 1, 0], u[0, 0, 1] = 512, 2.0 ** -8, 512
    a = torch.zeros(1, 2, 64, dtype=dtype)
    a[0, 0], a[0, 1] = 1, -1
    g = torch.zeros(rows, 40, dtype=dtype)
    g[:, 0], g[:, 1] = 1, -1
    y = m.adapted_linear(on, w, a.cuda(), u.cuda(), by, scale=256.0)
    (dx,) = torch.autograd.grad(y, on, g.cuda())
    assert (dx == -1).all()

# --------------------------------------------------------------------------
# Gradients asked for alone


def db_needs_no_rows(backward_weight, need, kept):
    """The bias's gradient of no rows' values: `x` (or what is kept of it) is not
    asked for. (On the CPU: a call that is refused for another reason.)"""
    from diff_gabor_splatting_amd import _native

    status = backward_weight(kept, need - 1)
    assert status == 4 and "workspace" in _native.lib.gs_last_error().decode()


def test_grouped_bias_gradient_takes_no_rows():
    from diff_gabor_splatting_amd import _native

    lib, p = _native.lib, ctypes.c_void_p(256)
    need = lib.gs_grouped_linear_backward_weight_workspace_size(0, 5000, 4, 64, 64)
    db_needs_no_rows(lambda x, size: lib.gs_grouped_linear_backward_weight(
        0, p, 64, x, 0, p, p, 5000, 4, 64, 64, None, p, p, size, None), need, None)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs,groups", [
    (900, 40, 24, 6), (3000, 300, 5, 4), (3000, 5, 300, 4), (700, 700, 130, 3),
    (130_000, 512, 512, 7), (3000, 1030, 40, 300)])
def test_grouped_bias_gradient_alone(dtype, rows, features, outputs, groups):
    """The sums of dy, whatever the shares; the rows are not kept for them."""
    m = layers()
    by, members = grouped_by(some_groups(rows, groups, 3), groups)
    x = normal(rows, features, seed=1, dtype=dtype).cuda()
    w = normal(groups, outputs, features, seed=2, dtype=dtype).cuda()
    b = normal(groups, outputs, seed=3, dtype=dtype).cuda().requires_grad_()
    g = normal(rows, outputs, seed=4, dtype=dtype)
    y = m.grouped_linear(x, w, by, b)
    x.mul_(2)  # raises in the backward pass where x is kept
    (got,) = torch.autograd.grad(y, b, g.cuda())
    want, size = (torch.stack([t.double()[at].sum(0) for at in members]) for t in (g, g.abs()))
    near(got, want, max(len(at) for at in members) * E * size, dtype)


def test_linear_bias_gradient_takes_no_rows():
    from diff_gabor_splatting_amd import _native

    lib, p = _native.lib, ctypes.c_void_p(256)
    need = lib.gs_linear_backward_weight_workspace_size(0, 5000, 64, 64)
    db_needs_no_rows(lambda kept, size: lib.gs_linear_backward_weight(
        0, p, 64, kept, kept, 5000, 64, 64, None, p, p, size, None), need, None)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs", [(900, 40, 24), (3000, 300, 5), (3000, 5, 300),
                                                   (700, 700, 130), (130_000, 512, 512)])
def test_shared_bias_gradient_alone(dtype, rows, features, outputs):
    """Of linear and of adapted_linear: the sums of dy, and nothing of the rows is
    kept for them."""
    m = layers()
    by, _ = grouped_by(some_groups(rows, 5, 3), 5)
    x = normal(rows, features, seed=1, dtype=dtype).cuda()
    w, b = normal(outputs, features, seed=2, dtype=dtype).cuda(), normal(outputs, seed=3,
                                                                       dtype=dtype).cuda()
    a, u = normal(5, 4, features, seed=5, dtype=dtype).cuda(), normal(5, outputs, 4, seed=6,
                                                                     dtype=dtype).cuda()
    g = normal(rows, outputs, seed=4, dtype=dtype)
    b.requires_grad_()
    before = torch.cuda.memory_allocated()
    y = m.linear(x, w, b)
    # (Memory is handed out in steps of 512 bytes.)
    assert torch.cuda.memory_allocated() - before < y.nbytes + rows * features
    z = m.adapted_linear(x, w, a, u, by, b)
    x.mul_(2)  # raises in the backward pass where x is kept
    for out in (y, z):
        (got,) = torch.autograd.grad(out, b, g.cuda())
        near(got, g.double().sum(0), rows * E * g.double().abs().sum(0), dtype)

# --------------------------------------------------------------------------
# Many rows: small whole numbers, whose sums float32 holds exactly in any order


def whole_numbers(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def whole(*shape, dtype):
        return torch.randint(-1, 2, shape, generator=gen, device="cuda").to(dtype)

    return whole


def rows_of(by, group, bounds):
    return by.order[bounds[group]:bounds[group + 1]].long()


@gpu_test
@pytest.mark.parametrize("dtype,rows,features,outputs,groups", [
    # The widest tiles of dW, 256 x 256: one with empty edges, several with
    # both edges ragged, and groups that end within a share.
    *((d, *size) for d in (torch.bfloat16, torch.float16)
      for size in ((600_001, 200, 200, 5), (100_003, 500, 508, 64), (60_000, 700, 508, 200))),
    # Parts joined by 64, 16 and 4 slices.
    *((d, 70_001, 40, 24, groups) for d in DTYPES for groups in (3, 6, 20))])
def test_grouped_linear_of_many_rows(dtype, rows, features, outputs, groups):
    m, whole = layers(), whole_numbers(rows + groups)
    x, g = whole(rows, features, dtype=dtype).requires_grad_(), whole(rows, outputs, dtype=dtype)
    w = whole(groups, outputs, features, dtype=dtype).requires_grad_()
    b = whole(groups, outputs, dtype=dtype).requires_grad_()
    by = m.row_groups(some_groups(rows, groups, 5, none=0.01).cuda(), groups)
    y = m.grouped_linear(x, w, by, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    bounds = by.offsets.tolist()
    for group in range(groups):
        at = rows_of(by, group, bounds)
        part, d, matrix = x[at].detach().double(), g[at].double(), w[group].detach().double()
        assert torch.equal(y[at], (part @ matrix.t() + b[group].double()).to(dtype))
        assert torch.equal(dx[at], (d @ matrix).to(dtype))
        assert torch.equal(dw[group], (d.t() @ part).to(dtype))
        assert torch.equal(db[group], d.sum(0).to(dtype))


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs,groups,rank", [
    (70_001, 40, 24, 3, 5),      # 64 slices
    (70_001, 40, 24, 12, 16),    # 16
    (70_001, 40, 24, 40, 33),    # 4
    (300_001, 72, 57, 7, 40),
    (300_001, 256, 136, 9, 64)])
def test_adapted_linear_of_many_rows(dtype, rows, features, outputs, groups, rank):
    """Inner values are whole halves below 2^15, which two parts hold."""
    m, whole = layers(), whole_numbers(rows + groups)
    x, g = whole(rows, features, dtype=dtype).requires_grad_(), whole(rows, outputs, dtype=dtype)
    w, b = whole(outputs, features, dtype=dtype), whole(outputs, dtype=dtype)
    a = whole(groups, rank, features, dtype=dtype).requires_grad_()
    u = whole(groups, outputs, rank, dtype=dtype).requires_grad_()
    by = m.row_groups(some_groups(rows, groups, 5, none=0.01).cuda(), groups)
    y = m.adapted_linear(x, w, a, u, by, b, scale=0.5)
    dx, da, du = torch.autograd.grad(y, (x, a, u), g)
    bounds = by.offsets.tolist()
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    shared = w.double()
    for group in range(groups):
        at = rows_of(by, group, bounds)
        inside[at] = True
        part, d = x[at].detach().double(), g[at].double()
        down, up = a[group].detach().double(), u[group].detach().double()
        inner, back = 0.5 * part @ down.t(), 0.5 * d @ up
        assert torch.equal(y[at], (part @ shared.t() + b.double() + inner @ up.t()).to(dtype))
        assert torch.equal(dx[at], (d @ shared + back @ down).to(dtype))
        assert torch.equal(da[group], (back.t() @ part).to(dtype))
        assert torch.equal(du[group], (d.t() @ inner).to(dtype))
    rest = ~inside
    assert torch.equal(y[rest], (x[rest].double() @ shared.t() + b.double()).to(dtype))
    assert torch.equal(dx[rest], (g[rest].double() @ shared).to(dtype))

# --------------------------------------------------------------------------
# Groups that change under a captured graph


@gpu_test
@pytest.mark.parametrize("dtype,rows", [(torch.bfloat16, 700), (torch.float32, 9000)])
def test_graphs_take_the_groups_of_each_replay(dtype, rows):
    """A captured launch holds any groups: each replay sorts the rows anew and
    goes by what it finds."""
    m = layers()
    x = normal(rows, 72, seed=1, dtype=dtype)
    w, b = normal(6, 64, 72, seed=2, dtype=dtype, scale=0.1), normal(6, 64, seed=3, dtype=dtype)
    shared, bias = normal(57, 64, seed=4, dtype=dtype, scale=0.1), normal(57, seed=5, dtype=dtype)
    down = normal(6, 8, 64, seed=6, dtype=dtype, scale=0.1)
    up = normal(6, 57, 8, seed=7, dtype=dtype, scale=0.3)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, shared, bias, down, up)]
    grad = normal(rows, 57, seed=8, dtype=dtype).cuda()
    index = some_groups(rows, 6, 9).cuda()

    def step(index):
        x, w, b, shared, bias, down, up = leaves
        by = m.row_groups(index, 6)
        h = m.grouped_linear(x, w, by, b)
        y = m.adapted_linear(h, shared, down, up, by, bias, scale=0.5)
        grads = torch.autograd.grad(y, leaves, grad)
        return (y.detach(), h.detach(), by.order, by.offsets, *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(index)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(index)
    all_rows = torch.full((rows,), 4)
    uneven = torch.where(torch.arange(rows) == 17, 5, 0)
    for other in (some_groups(rows, 6, 10), all_rows, all_rows - 5, torch.arange(rows) % 6, uneven,
                  some_groups(rows, 6, 9)):
        index.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step(index.clone())):
            assert torch.equal(got, want)

# --------------------------------------------------------------------------
# Memory beside the results

SENTINEL, MARGIN = 0x5A, 1 << 16


class Guarded:
    """`count` bytes between margins that a call must leave as they are."""

    def __init__(self, count):
        self.count = count
        self.all = torch.full((count + 2 * MARGIN,), SENTINEL, dtype=torch.uint8, device="cuda")

    @property
    def pointer(self):
        return ctypes.c_void_p(self.all.data_ptr() + MARGIN)

    def intact(self):
        return bool((self.all[:MARGIN] == SENTINEL).all()) and \
            bool((self.all[MARGIN + self.count:] == SENTINEL).all())


def malformed_groups(rows, groups):
    """Offsets that fall, pass the rows or are below zero, and places that are
    not rows."""
    gen = torch.Generator().manual_seed(rows + groups)
    wild = lambda *shape: torch.randint(-(1 << 31), 1 << 31, shape, generator=gen)  # noqa: E731
    near_by = lambda *shape: torch.randint(-40, rows + 40, shape, generator=gen)  # noqa: E731
    for offsets in (wild(groups + 1), near_by(groups + 1), near_by(groups + 1).sort().values,
                    near_by(groups + 1).sort(descending=True).values,
                    torch.full((groups + 1,), rows), torch.full((groups + 1,), 1 << 30)):
        for order in (None, wild(rows), near_by(rows)):
            yield (offsets.to(torch.int32).cuda(),
                   None if order is None else order.to(torch.int32).cuda())


@gpu_test
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,features,outputs,groups,rank", [
    (12, 72, 57, 6, 8), (700, 72, 57, 6, 8), (700, 72, 130, 130, 40), (3000, 1100, 40, 5, 8),
    (3000, 40, 1100, 5, 33)])
def test_wrong_groups_write_nothing_beside_the_results(dtype, rows, features, outputs, groups, rank):
    """The C entry points with groups that are none: what is written is the
    results, the inner rows and the workspace."""
    from diff_gabor_splatting_amd import _native

    lib, size = _native.lib, 4 if dtype == 0 else 2
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    held = {name: torch.zeros(count * size, dtype=torch.uint8, device="cuda") for name, count in (
        ("x", rows * features), ("g", rows * outputs), ("w", groups * outputs * features),
        ("b", groups * outputs), ("down", groups * rank * features),
        ("up", groups * outputs * rank))}
    p = {name: ctypes.c_void_p(t.data_ptr()) for name, t in held.items()}
    inner_size = lib.gs_adapted_linear_inner_size(rows, rank)
    sum_size = lib.gs_grouped_linear_backward_weight_workspace_size(dtype, rows, groups, features,
                                                                    outputs)
    narrow_size = lib.gs_adapted_linear_backward_adapters_workspace_size(rows, groups, features,
                                                                         outputs, rank)
    for offsets, order in malformed_groups(rows, groups):
        at = ctypes.c_void_p(offsets.data_ptr())
        by = None if order is None else ctypes.c_void_p(order.data_ptr())
        y, dx, z, dz = (Guarded(rows * n * size) for n in (outputs, features, outputs, features))
        dw, db = Guarded(groups * outputs * features * size), Guarded(groups * outputs * size)
        da, du = Guarded(groups * rank * features * size), Guarded(groups * outputs * rank * size)
        inner, back = Guarded(inner_size), Guarded(inner_size)
        sums, narrow = Guarded(sum_size), Guarded(narrow_size)
        calls = (
            lib.gs_grouped_linear_forward(dtype, p["x"], features, p["w"], p["b"], by, at, rows,
                                          groups, features, outputs, y.pointer, stream),
            lib.gs_grouped_linear_backward_input(dtype, p["g"], outputs, p["w"], by, at, rows, groups,
                                                 features, outputs, dx.pointer, stream),
            lib.gs_grouped_linear_backward_weight(
                dtype, p["g"], outputs, p["x"], features, by, at, rows, groups, features, outputs,
                dw.pointer, db.pointer, sums.pointer, sum_size, stream),
            lib.gs_adapted_linear_forward(
                dtype, p["x"], features, p["w"], p["b"], p["down"], p["up"], 0.5, by, at, rows,
                groups, features, outputs, rank, inner.pointer, inner_size, z.pointer, stream),
            lib.gs_adapted_linear_backward_input(
                dtype, p["g"], outputs, p["w"], p["down"], p["up"], 0.5, by, at, rows, groups,
                features, outputs, rank, back.pointer, inner_size, dz.pointer, stream),
            lib.gs_adapted_linear_backward_adapters(
                dtype, p["g"], outputs, p["x"], features, inner.pointer, back.pointer, by, at, rows,
                groups, features, outputs, rank, da.pointer, du.pointer, narrow.pointer, narrow_size,
                stream))
        assert calls == (0,) * 6, lib.gs_last_error()
        torch.cuda.synchronize()
        for name, buffer in dict(y=y, dx=dx, z=z, dz=dz, dw=dw, db=db, da=da, du=du, inner=inner,
                                 back=back, sums=sums, narrow=narrow).items():
            assert buffer.intact(), name
