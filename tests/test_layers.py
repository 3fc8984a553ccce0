"""The decoder layers against their formulas in 64 bits (oracle/layers.py).

CPU: the 8-bit form's definition, argument errors of the C entry points and
of the Python functions. GPU: every operator over types, widths, row counts,
strides and special values.

Tolerances are worst-case rounding bounds. With u the unit roundoff of the
output type (2^-8 bfloat16, 2^-11 float16, 2^-24 float32; half a unit in the
last place, relative) and e = 2^-24, an output that is computed in float32
and rounded once is off by at most u |out| + the float32 error, and a
float32 sum of n terms t by at most n e sum |t|.
"""

import ctypes
import math

import pytest
import torch

from oracle import layers as oracle

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
E = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Below a type's normal range the spacing is fixed: half of it.
FLOOR = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def layers():
    from diff_gabor_splatting_amd import layers as module

    return module


def generator(seed):
    return torch.Generator().manual_seed(seed)


def normal(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=generator(seed)) * scale).to(dtype)


def near(got, expected, error, dtype):
    """|got - expected| <= rounding to dtype + the float32 error, everywhere."""
    got = got.detach().cpu().double()
    assert got.shape == expected.shape
    bound = UNIT[dtype] * (expected.abs() + error) + error + FLOOR[dtype]
    off = (got - expected).abs()
    worst = (off / bound).max().item() if got.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{worst:.3g} times the bound"


# --------------------------------------------------------------------------
# CPU


def test_oracle_kept_is_the_first_exponent_that_is_enough():
    x = torch.tensor([[127.5, 1.0] + [0.0] * 30, [127.49, -63.5] + [0.0] * 30,
                      [0.0] * 32, [64.0, 0.5] + [0.0] * 30])
    q, b, v = oracle.kept(x)
    assert b[:, 0].tolist() == [128, 127, 1, 127]
    assert q[0, :2].tolist() == [64, 0]      # 127.5 / 2 and 1 / 2, ties to even
    assert q[1, :2].tolist() == [127, -64]   # 63.5 to the even 64
    assert q[3, :2].tolist() == [64, 0]
    assert v[0, 0] == 128 and v[2].abs().max() == 0


def test_oracle_kept_error_is_within_a_step():
    x = normal(50, 100, seed=3)
    _, _, v = oracle.kept(x)
    groups = torch.nn.functional.pad(x, (0, 28)).view(50, 4, 32).abs().amax(-1)
    limit = groups.repeat_interleave(32, 1)[:, :100].double() / 127
    assert ((v - x.double()).abs() <= limit).all()


def test_oracle_gradients_match_autograd():
    x, g = normal(6, 40, seed=4).double(), normal(6, 40, seed=5).double()
    w, b = normal(40, seed=6).double(), normal(40, seed=7).double()
    for t in (x, w, b):
        t.requires_grad_()
    y = torch.nn.functional.layer_norm(x, (40,), w, b)
    expected = torch.autograd.grad(y, (x, w, b), g)
    dx, dw, db, _, _ = oracle.layer_norm_backward(x.detach(), g, w.detach())
    torch.testing.assert_close(oracle.layer_norm(x, w, b)[0], y)
    for got, want in zip((dx, dw, db), expected):
        torch.testing.assert_close(got, want)
    for kind, function in (("gelu", torch.nn.functional.gelu), ("silu", torch.nn.functional.silu),
                           ("sine", lambda z: torch.sin(30 * z))):
        y = function(x)
        torch.testing.assert_close(oracle.activation(x, kind, 30.0), y)
        torch.testing.assert_close(oracle.slope(x, kind, 30.0),
                                   torch.autograd.grad(y.sum(), x)[0])


def test_c_entry_points_refuse_bad_arguments():
    from diff_gabor_splatting_amd import _native

    lib, p = _native.lib, ctypes.c_void_p(256)

    def refused(status, code, text):
        assert status == code and text in lib.gs_last_error().decode(), lib.gs_last_error()

    refused(lib.gs_checkpoint8_write(3, p, 8, 1, 8, p, p, None), 1, "unknown type")
    refused(lib.gs_checkpoint8_write(0, p, 8, -1, 8, p, p, None), 1, "negative")
    refused(lib.gs_checkpoint8_write(0, p, 8, 1, 0, p, p, None), 1, "features")
    refused(lib.gs_checkpoint8_write(0, p, 7, 2, 8, p, p, None), 1, "overlap")
    refused(lib.gs_checkpoint8_write(0, p, 8, 1 << 60, 8, p, p, None), 2, "too many rows")
    refused(lib.gs_checkpoint8_write(0, None, 8, 1, 8, p, p, None), 1, "null")
    refused(lib.gs_checkpoint8_read(0, p, None, 1, 8, p, None), 1, "null")
    refused(lib.gs_activation_forward(0, 9, 1.0, p, 8, 1, 8, p, p, p, None), 1, "activation")
    refused(lib.gs_activation_forward(0, 0, math.inf, p, 8, 1, 8, p, p, p, None), 1, "omega")
    refused(lib.gs_activation_forward(0, 0, 1.0, p, 8, 1, 8, p, p, None, None), 1, "null")
    refused(lib.gs_activation_backward(0, 0, 1.0, p, 8, None, p, 1, 8, p, None), 1, "null")
    refused(lib.gs_layer_norm_forward(1, 2, p, 8, p, p, 1e-5, 1, 8, p, p, None, None, None), 1,
            "parameters")
    refused(lib.gs_layer_norm_forward(0, 0, p, 8, p, p, -1.0, 1, 8, p, p, None, None, None), 1,
            "eps")
    refused(lib.gs_layer_norm_forward(0, 0, p, 16385, p, p, 1e-5, 1, 16385, p, p, None, None,
                                      None), 1, "at most 16384")
    refused(lib.gs_layer_norm_forward(0, 0, p, 8, p, p, 1e-5, 1, 8, p, None, p, p, None), 1,
            "null")
    # Either x or what was kept, and a workspace for the parameters' gradients.
    refused(lib.gs_layer_norm_backward(0, 0, p, 8, p, 8, p, p, p, p, 1, 8, p, p, p, p, 1 << 20,
                                       None), 1, "null")
    need = lib.gs_layer_norm_backward_workspace_size(100, 8)
    refused(lib.gs_layer_norm_backward(0, 0, p, 8, p, 8, None, None, p, p, 100, 8, p, p, p, p,
                                       need - 1, None), 4, "workspace")
    refused(lib.gs_linear_forward(0, p, 8, None, None, 1, 8, 8, p, None, None, None), 1, "null")
    refused(lib.gs_linear_forward(0, p, 8, p, None, 1, 8, 0, p, None, None, None), 1, "features")
    refused(lib.gs_linear_forward(0, p, 8, p, None, 1, 8, 1 << 20, p, None, None, None), 1,
            "at most")
    refused(lib.gs_linear_backward_input(0, p, 3, p, 2, 8, 4, p, None), 1, "overlap")
    need = lib.gs_linear_backward_weight_workspace_size(0, 100, 8, 4)
    assert need > 0
    refused(lib.gs_linear_backward_weight(0, p, 4, p, p, 100, 8, 4, p, p, p, need - 1, None), 4,
            "workspace")
    # No rows: nothing to do and nothing touched.
    assert lib.gs_checkpoint8_write(0, None, 8, 0, 8, None, None, None) == 0
    assert lib.gs_linear_forward(0, None, 8, None, None, 0, 8, 8, None, None, None, None) == 0
    assert lib.gs_last_error() == b""


def test_python_functions_refuse_cpu_tensors_and_bad_options():
    m = layers()
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    for call in (lambda: m.quantize(x), lambda: m.activation(x), lambda: m.layer_norm(x),
                 lambda: m.linear(x, w)):
        with pytest.raises(ValueError, match="on a HIP device"):
            call()
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        m.quantize([1.0])
    with pytest.raises(TypeError, match="must be a Checkpoint"):
        m.dequantize(x)
    with pytest.raises(ValueError, match="kind must be one of"):
        m.activation(x, "tanh")
    with pytest.raises(ValueError, match="omega"):
        m.activation(x, omega=math.nan)
    with pytest.raises(ValueError, match="checkpoint must be"):
        m.layer_norm(x, checkpoint="4bit")
    with pytest.raises(ValueError, match="eps"):
        m.layer_norm(x, eps=-1.0)


def layer_calls(device="cpu"):
    """Each operator as a function of the rows alone, by name."""
    m = layers()
    w, b = torch.ones(8, device=device), torch.zeros(8, device=device)
    big, four = torch.ones(4, 8, device=device), torch.zeros(4, device=device)
    return {"activation": lambda t: m.activation(t),
            "layer_norm": lambda t: m.layer_norm(t, w, b),
            "linear": lambda t: m.linear(t, big, four)}


def refuses_what_would_lose_a_result(calls, x):
    """Forward mode and the tracers follow torch's operators, not these
    calls: without a refusal a tangent is lost and a replayed trace returns
    memory that nothing has written."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, call in calls.items():
        for t in (x, x.clone().requires_grad_()):
            for trace in (lambda: torch.jit.trace(call, (t,)), lambda: make_fx(call)(t),
                          lambda: make_fx(call, pre_dispatch=True)(t),
                          lambda: make_fx(call, tracing_mode="fake")(t)):
                with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                    trace()
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode"):
                call(dual)


def test_forward_mode_and_tracing_are_refused():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    m = layers()
    x = torch.zeros(2, 8)
    refuses_what_would_lose_a_result(layer_calls(), x)
    with forward_ad.dual_level():
        w = forward_ad.make_dual(torch.ones(8), torch.ones(8))
        big = forward_ad.make_dual(torch.ones(4, 8), torch.ones(4, 8))
        for call in (lambda: m.layer_norm(x, w), lambda: m.layer_norm(x, None, w),
                     lambda: m.linear(x, big), lambda: m.linear(x, torch.ones(8, 8), w)):
            with pytest.raises(RuntimeError, match="no forward-mode"):
                call()
    kept = m.Checkpoint(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8),
                        x.shape, x.dtype)
    for name, trace in (("quantize", lambda: make_fx(lambda t: m.quantize(t).values)(x)),
                        ("dequantize", lambda: torch.jit.trace(
                            lambda t: t + m.dequantize(kept), (x,)))):
        with pytest.raises(RuntimeError, match=f"^{name} cannot be traced"):
            trace()
    # Outside of them the refusal leaves no trace.
    with pytest.raises(ValueError, match="on a HIP device"):
        m.activation(x)


def test_learned_numbers_are_refused():
    """omega and eps have no gradient: one that asks for it would get none."""
    m = layers()
    x, learned = torch.zeros(2, 8), torch.tensor(30.0, requires_grad=True)
    with pytest.raises(ValueError, match="omega has no gradient"):
        m.activation(x, "sine", learned)
    with pytest.raises(ValueError, match="eps has no gradient"):
        m.layer_norm(x, eps=learned)
    with pytest.raises(ValueError, match="on a HIP device"):
        m.activation(x, "sine", learned.detach())


# --------------------------------------------------------------------------
# GPU: the 8-bit form


def gpu_test(function):
    for mark in gpu:
        function = mark(function)
    return function


def same_bytes(x, dtype):
    m = layers()
    kept = m.quantize(x.cuda())
    q, b, v = oracle.kept(x.reshape(-1, x.shape[-1]))
    assert torch.equal(kept.values.cpu(), q) and torch.equal(kept.exponents.cpu(), b)
    back = m.dequantize(kept)
    assert back.dtype == dtype and back.shape == x.shape
    assert torch.equal(back.cpu().double().nan_to_num(7e77),
                       v.reshape(x.shape).nan_to_num(7e77))


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 8), (7, 40), (7, 187),
                                   (1000, 64), (513, 1000), (2, 3, 5, 96), (30000, 96),
                                   (40000, 100)])
def test_checkpoint_bytes(dtype, shape):
    same_bytes(normal(*shape, seed=sum(shape), dtype=dtype, scale=3.0), dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_of_special_values(dtype):
    most = torch.finfo(dtype).max
    rows = [[0.0], [-0.0, 1.0], [most, -most, most / 3], [most / 1.01], [2.0 ** -24, 2.0 ** -20],
            [torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 4], [127.5, 0.25, 0.75],
            [127.0, 63.5, 62.5, -0.5, 1.5], [127.49, 2.5], [math.inf, 1.0], [1.0, math.nan],
            [-math.inf, math.inf], [1e-6, 1.0], [255.0], [254.9, 3.0]]
    x = torch.zeros(len(rows), 70)
    for i, row in enumerate(rows):
        x[i, :len(row)] = torch.tensor(row)
        x[i, 40:40 + len(row)] = torch.tensor(row) / 3
    same_bytes(x.to(dtype), dtype)


@gpu_test
def test_checkpoint_reads_back_in_another_type():
    m = layers()
    x = normal(9, 50, seed=1, dtype=torch.bfloat16)
    _, _, v = oracle.kept(x)
    assert torch.equal(m.dequantize(m.quantize(x.cuda()), torch.float32).cpu().double(), v)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_of_strided_rows(dtype):
    m = layers()
    base = normal(12, 4, 200, seed=2, dtype=dtype)
    views = {
        "rows apart": lambda t: t[:, 1, :96],
        "misaligned": lambda t: t[:, 2, 3:100],
        "collapsing": lambda t: t[..., :64],
        "not collapsing": lambda t: t[:, :3, 8:72],
        "transposed": lambda t: t.transpose(0, 2),
        "expanded": lambda t: t[:1, 0, :40].expand(6, 40),
        "one feature": lambda t: t[:, :, :1],
        "vector": lambda t: t[3, 1],
        "every second": lambda t: t[:, 0, ::2],
    }
    for name, view in views.items():
        got = m.quantize(view(base.cuda()))
        want = view(base)
        q, b, _ = oracle.kept(want.reshape(-1, want.shape[-1]))
        assert torch.equal(got.values.cpu(), q) and torch.equal(got.exponents.cpu(), b), name


# --------------------------------------------------------------------------
# GPU: activations


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["sine", "gelu", "silu"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 57), (64, 128), (5, 1000), (2, 4, 40), (9000, 256)])
def test_activation(dtype, kind, shape):
    m = layers()
    scale = 0.2 if kind == "sine" else 3.0
    x = normal(*shape, seed=11, dtype=dtype, scale=scale)
    g = normal(*shape, seed=12, dtype=dtype)
    on = x.cuda().requires_grad_()
    y = m.activation(on, kind)
    (dx,) = torch.autograd.grad(y, on, g.cuda())
    z = oracle.kept(x.reshape(-1, shape[-1]))[2].reshape(shape)
    want, slope = oracle.activation(x, kind, 30.0), oracle.slope(z, kind, 30.0)
    # sine: the phase's fraction and the polynomial to a few units of 2^-24
    # of their largest value; gelu: 1.5e-7 on erf (half of that on Phi), the
    # hardware's exp2 and reciprocal; silu: the same two.
    error = {"sine": 16 * E, "gelu": 8e-8 + 16 * E, "silu": 16 * E}[kind]
    size = 1.0 if kind == "sine" else 1 + x.double().abs()
    near(y, want, error * size, dtype)
    wide = 30.0 if kind == "sine" else 1 + z.abs() + z * z
    near(dx, g.double() * slope, g.double().abs() * error * wide, dtype)
    # Without a gradient nothing is kept and the values are the same.
    assert torch.equal(m.activation(x.cuda(), kind), y.detach())


def float32_activation(kind, x):
    """(value, its 64-bit value, slope, its 64-bit value) of float32 rows; the
    slope is that at the kept rows."""
    m = layers()
    on = x.cuda().requires_grad_()
    y = m.activation(on, kind)
    (dx,) = torch.autograd.grad(y, on, torch.ones_like(y))
    z = oracle.kept(x)[2]
    return (y.detach().cpu().double(), oracle.activation(x, kind, 30.0), dx.cpu().double(),
            oracle.slope(z, kind, 30.0))


def relative_rms(got, want):
    return ((got - want).norm() / want.norm()).item()


@gpu_test
@pytest.mark.parametrize("scale", [1 / 30, 1.0, 30.0])
def test_float32_sine_is_as_exact_as_its_type(scale):
    """Two roundings, the phase's and the function's, at phases of 1, 30 and
    900: an rms of 2^-24 times the root of two thirds of the largest value a
    rounding error is half a unit of."""
    y, value, dx, slope = float32_activation("sine", normal(512, 256, seed=18, scale=scale))
    assert relative_rms(y, value) <= E * (2 / 3) ** 0.5
    assert relative_rms(dx, slope) <= E * (2 / 3) ** 0.5


@gpu_test
@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_float32_gelu_is_as_exact_as_its_type(scale):
    """A rounding is off by half a unit, 2^-24, at most, with an rms of a
    root of three less: rms relative error of three roundings (the
    function's, Phi's, its polynomial's). The negative tail, where the value
    is the product of z, a polynomial and the bell: by value, the units of
    2^-24 of its operations (exp2 2, reciprocal and its argument 3, the
    polynomial's last steps 2, the bell's correction 1, three products 3) and
    one for the rest."""
    y, value, dx, slope = float32_activation("gelu", normal(512, 256, seed=15, scale=scale))
    assert relative_rms(y, value) <= E
    assert relative_rms(dx, slope) <= E
    x = -2 - 4 * torch.rand(64, 256, generator=generator(16))
    y, value, _, _ = float32_activation("gelu", x)
    assert ((y - value).abs() <= 12 * E * value.abs()).all()


@gpu_test
@pytest.mark.parametrize("scale", [1.0, 4.0])
def test_float32_silu_is_as_exact_as_its_type(scale):
    """rms as for the sine: two roundings (the sum 1 + exp and the quotient).
    Where the exponential is all of the sum, by value, in units of 2^-24:
    exp2 2, its correction 1, the sum 1, the quotient 2."""
    y, value, _, _ = float32_activation("silu", normal(512, 256, seed=19, scale=scale))
    assert relative_rms(y, value) <= E * (2 / 3) ** 0.5
    x = -2 - 60 * torch.rand(64, 256, generator=generator(20))
    y, value, _, _ = float32_activation("silu", x)
    assert ((y - value).abs() <= 6 * E * value.abs()).all()


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_keeps_its_tail_in_two_bytes(dtype):
    """Phi(-|z|) to 1.2e-5 of itself (the fit), the bell's argument (up to 26,
    rounded twice) 2.2e-6, a dozen float32 roundings below 1e-6: 2e-5 in all,
    and then the one rounding to the type."""
    m = layers()
    x = (-2 - 4 * torch.rand(64, 256, generator=generator(17))).to(dtype)
    on = x.cuda().requires_grad_()
    y = m.activation(on, "gelu")
    (dx,) = torch.autograd.grad(y, on, torch.ones_like(y))
    value = oracle.activation(x, "gelu", 0.0)
    near(y, value, 2e-5 * value.abs(), dtype)
    z = oracle.kept(x)[2]
    near(dx, oracle.slope(z, "gelu", 0.0),
         2e-5 * torch.special.ndtr(z) + 4e-6 * z.abs() * torch.exp(-z * z / 2) * 0.4, dtype)


@gpu_test
def test_activation_of_special_values():
    m = layers()
    x = torch.zeros(4, 64)
    x[0, 0], x[1, 40], x[2, 3] = math.inf, -math.inf, math.nan
    x[3, :4] = torch.tensor([1e30, -1e30, 88.0, -88.0])
    for kind in ("gelu", "silu"):
        on = x.cuda().requires_grad_()
        y = m.activation(on, kind)
        (dx,) = torch.autograd.grad(y, on, torch.ones_like(y))
        assert y[0, 0] == math.inf and y[2, 3].isnan()
        torch.testing.assert_close(y[3, :4].cpu(), torch.tensor([1e30, 0.0, 88.0, 0.0]),
                                   atol=1e-30, rtol=1e-6)
        # The whole group of a non-finite input has no derivative, no other.
        lost = dx.isnan().cpu()
        expected = torch.zeros(4, 64, dtype=torch.bool)
        expected[0, :32] = expected[1, 32:] = expected[2, :32] = True
        assert torch.equal(lost, expected)


@gpu_test
def test_sine_of_large_phases():
    """The phase's fraction is taken without rounding the phase: at phases of
    thousands the sine is as exact as at small ones."""
    m = layers()
    x = normal(64, 64, seed=13, scale=300.0)
    y = m.activation(x.cuda(), "sine", 30.0).cpu().double()
    assert (y - torch.sin(30 * x.double())).abs().max() < 1e-6


@gpu_test
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sine_of_phases_past_whole_floats(dtype):
    """Past 2^24 revolutions the rounded product with omega / 2 pi is whole,
    and what it lacks is more than half a revolution. The fraction is off by
    at most 2^-48 of the revolutions (omega / 2 pi as two floats: 2^-49; the
    sum of the two small products, at most 2^-24 of the revolutions: 2^-49);
    twice that is allowed. A sine stays a sine, whatever its phase."""
    m = layers()
    for size in (1e5, 1e7, 1e9, 1e12, 1e20, 1e30):
        x = (normal(32, 64, seed=14) * size).to(dtype)
        on = x.cuda().requires_grad_()
        y = m.activation(on, "sine", 30.0)
        (dx,) = torch.autograd.grad(y, on, torch.ones_like(y))
        y, dx = y.detach().cpu().double(), dx.cpu().double()
        assert y.abs().max() <= 1 + 1e-6 and dx.abs().max() <= 30 * (1 + 1e-6)
        turns = 30 * x.double().abs() / (2 * math.pi)
        error = 2 * math.pi * turns * 2.0 ** -47
        near(y.to(dtype), oracle.activation(x, "sine", 30.0), error + 16 * E, dtype)
        z = oracle.kept(x)[2]
        near(dx.to(dtype), oracle.slope(z, "sine", 30.0),
             30 * (2 * math.pi * 30 * z.abs() / (2 * math.pi) * 2.0 ** -47 + 16 * E), dtype)


# --------------------------------------------------------------------------
# GPU: layer norm


def norm_case(shape, dtype, weights, eight, seed=21, parameters=True, offset=0.5):
    m = layers()
    features = shape[-1]
    x = (normal(*shape, seed=seed) + offset * normal(*shape[:-1], 1, seed=seed + 1)).to(dtype)
    g = normal(*shape, seed=seed + 2, dtype=dtype)
    w = (1 + 0.1 * normal(features, seed=seed + 3)).to(weights) if parameters else None
    b = normal(features, seed=seed + 4, dtype=weights) if parameters else None
    inputs = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    y = m.layer_norm(*inputs, checkpoint="8bit" if eight else "full")
    grads = torch.autograd.grad(y, inputs, g.cuda())
    check_norm(x.reshape(-1, features), g.reshape(-1, features), w, b, eight,
               y.reshape(-1, features), [grads[0].reshape(-1, features), *grads[1:]])
    with torch.no_grad():
        assert torch.equal(m.layer_norm(*inputs), y)


def check_norm(x, g, w, b, eight, y, grads, eps=1e-5):
    rows, features = x.shape
    dtype = x.dtype
    want, h, r = oracle.layer_norm(x, w, b, eps)
    # A lane adds at most 32 values in turn and then the lanes', 6 + 16 steps:
    # the mean is off by n e of the mean magnitude, the variance, its root and
    # h by as much relatively.
    n = 64
    size = x.double().abs().amax(1, keepdim=True) * r
    spread = n * E * (size + h.abs())
    scale = 1.0 if w is None else w.double().abs()
    near(y, want, spread * scale + 4 * E * want.abs(), dtype)
    dx, dw, db, h, r = oracle.layer_norm_backward(x, g, w, eps, eight)
    a = g.double().abs() * scale
    along = (a * h.abs()).mean(1, keepdim=True)
    error = r * (n * E * (a + a.mean(1, keepdim=True) + h.abs() * along)
                 + spread * along + h.abs() * (a * spread).mean(1, keepdim=True))
    near(grads[0], dx, error, dtype)
    if w is not None:
        terms = n + rows / 16
        near(grads[1], dw, (g.double().abs() * (terms * E * h.abs() + spread)).sum(0), w.dtype)
        near(grads[2], db, terms * E * g.double().abs().sum(0), w.dtype)


@gpu_test
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("features", [1, 7, 8, 31, 33, 64, 96, 187, 256, 512, 513, 520, 1000, 1024,
                                      2048, 2056, 4099, 8192, 8200, 16384])
def test_layer_norm_widths(features, eight):
    # One feature leaves h = 0 and no variance: eps alone sets r.
    norm_case((5, features), torch.float32, torch.float32, eight)
    norm_case((67, features), torch.bfloat16, torch.bfloat16, eight, seed=31)


@gpu_test
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype,weights", [(torch.float32, torch.float32),
                                           (torch.bfloat16, torch.float32),
                                           (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float32),
                                           (torch.float16, torch.float16)])
@pytest.mark.parametrize("shape", [(1, 64), (2, 3, 5, 48), (4099, 40), (20011, 72)])
def test_layer_norm(dtype, weights, eight, shape):
    norm_case(shape, dtype, weights, eight)


@gpu_test
@pytest.mark.parametrize("eight", [False, True])
def test_layer_norm_without_parameters_and_with_a_large_mean(eight):
    norm_case((33, 128), torch.float32, torch.float32, eight, parameters=False)
    norm_case((33, 128), torch.float32, torch.float32, eight, offset=300.0)


@gpu_test
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("features", [5, 57, 187, 500, 1000, 4099, 16384])
def test_layer_norm_of_constant_rows(features, eight):
    """A row of one value is its own mean to the last bit, whatever the value:
    the output is the bias, h and with it dw are zero. Rows whose spread is a
    few units of the mean's last place: the mean is off by half a unit and
    what the n differences' sum loses, n 2^-24 of their size."""
    m = layers()
    at = torch.tensor([4097.3, 1000.1, -33333.3, 0.1, 1e-20, 1e20, 0.0])
    x = at[:, None].expand(-1, features).contiguous()
    w, b, g = normal(features, seed=61), normal(features, seed=62), normal(7, features, seed=63)
    inputs = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = m.layer_norm(*inputs, checkpoint="8bit" if eight else "full")
    dx, dw, db = torch.autograd.grad(y, inputs, g.cuda())
    assert torch.equal(y.detach().cpu(), b.expand(7, -1))
    assert torch.equal(dw.cpu(), torch.zeros(features))
    unit = 2.0 ** -11  # of 4097.3
    x = 4097.3 + unit * torch.randint(-8, 9, (40, features), generator=generator(64))
    eps = 1.0  # the differences stay below it: r is 1 to 2^-14
    y = m.layer_norm(x.cuda(), eps=eps).cpu().double()
    want = oracle.layer_norm(x, eps=eps)[0]
    assert ((y - want).abs() <= unit * (0.5 + 16 * features * E) + 2 * E).all()


@gpu_test
def test_layer_norm_of_one_parameter():
    m = layers()
    x, w = normal(9, 48, seed=1).cuda(), normal(48, seed=2).cuda()
    g = normal(9, 48, seed=3).cuda()
    for name, other in (("weight", "bias"), ("bias", "weight")):
        p = w.clone().requires_grad_()
        y = m.layer_norm(x, **{name: p})
        (got,) = torch.autograd.grad(y, p, g)
        both = {name: w.clone().requires_grad_(),
                other: (torch.ones_like(w) if other == "weight" else torch.zeros_like(w))}
        z = m.layer_norm(x, **both)
        assert torch.equal(y, z)
        assert torch.equal(got, torch.autograd.grad(z, both[name], g)[0])


@gpu_test
@pytest.mark.parametrize("eight", [False, True])
def test_layer_norm_keeps_a_bad_row_to_itself(eight):
    """Rows with NaN or infinities give NaN in their own outputs and input
    gradients, and leave other rows' untouched; a constant row is all bias."""
    m = layers()
    x = normal(40, 96, seed=5)
    bad = x.clone()
    bad[3, 7], bad[20, 95], bad[39, 0] = math.nan, math.inf, -math.inf
    bad[10] = 0.25
    x[10] = 0.25
    w, b, g = normal(96, seed=6), normal(96, seed=7), normal(40, 96, seed=8)
    outs = []
    for t in (x, bad):
        inputs = [v.cuda().requires_grad_() for v in (t, w, b)]
        y = m.layer_norm(*inputs, checkpoint="8bit" if eight else "full")
        outs.append((y, torch.autograd.grad(y, inputs, g.cuda())))
    rows = torch.ones(40, dtype=torch.bool)
    rows[[3, 20, 39]] = False
    assert torch.equal(outs[0][0][rows.cuda()], outs[1][0][rows.cuda()])
    assert torch.equal(outs[0][1][0][rows.cuda()], outs[1][1][0][rows.cuda()])
    assert outs[1][0][~rows.cuda()].isnan().all() and outs[1][1][0][~rows.cuda()].isnan().all()
    assert torch.equal(outs[1][0][10].cpu(), b)
    assert torch.equal(outs[0][1][2], outs[1][1][2])  # the bias's gradient reads dy alone


# --------------------------------------------------------------------------
# GPU: linear layers


def linear_case(shape, outputs, dtype, bias=True, seed=41):
    m = layers()
    features = shape[-1]
    x = normal(*shape, seed=seed, dtype=dtype)
    w = normal(outputs, features, seed=seed + 1, dtype=dtype, scale=features ** -0.5)
    b = normal(outputs, seed=seed + 2, dtype=dtype) if bias else None
    g = normal(*shape[:-1], outputs, seed=seed + 3, dtype=dtype)
    inputs = [t.cuda().requires_grad_() for t in (x, w, b) if t is not None]
    y = m.linear(*inputs)
    grads = torch.autograd.grad(y, inputs, g.cuda())
    with torch.no_grad():
        assert torch.equal(m.linear(*inputs), y)
    assert y.shape == (*shape[:-1], outputs) and grads[0].shape == shape
    x, g = x.reshape(-1, features), g.reshape(-1, outputs)
    rows = x.shape[0]
    size = oracle.linear(x.abs(), w.abs(), None if b is None else b.abs())
    near(y.reshape(rows, outputs), oracle.linear(x, w, b), (features + 2) * E * size, dtype)
    dx, dw, db = oracle.linear_backward(x, w, g)
    near(grads[0].reshape(rows, features), dx,
         (outputs + 2) * E * (g.double().abs() @ w.double().abs()), dtype)
    held = oracle.kept(x)[2].abs()
    near(grads[1], dw, (rows + 2) * E * (g.double().abs().t() @ held), dtype)
    if bias:
        near(grads[2], db, (rows + 2) * E * g.double().abs().sum(0), dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs", [
    (1, 1, 1), (1, 64, 64), (1, 1000, 57), (2, 33, 18), (5, 8, 8), (16, 128, 128), (17, 31, 129),
    (64, 96, 57), (127, 130, 63), (128, 64, 256), (129, 256, 130), (300, 187, 18),
    (1000, 40, 72), (2500, 264, 136)])
def test_linear(dtype, rows, features, outputs):
    linear_case((rows, features), outputs, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_shapes_and_no_bias(dtype):
    linear_case((2, 3, 4, 48), 24, dtype)
    linear_case((40,), 24, dtype)
    linear_case((50, 64), 32, dtype, bias=False)


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,outputs", [
    (140, 1100, 40), (140, 40, 1100), (130, 1030, 1030), (6, 24, 4200), (6, 4200, 24),
    (3, 1500, 130), (33, 512, 512), (4000, 512, 130), (2000, 130, 512), (3000, 70, 130)])
def test_linear_wide(dtype, rows, features, outputs):
    """Matrices with a side longer than the streaming kernel takes, panels of
    every width, and tiles of dW of every shape."""
    linear_case((rows, features), outputs, dtype)


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_of_many_rows(dtype):
    """Rows enough for the widest tiles of dW (2e10 and 1e10 products), against
    the sum over parts of the rows, whose bound the parts' sizes give."""
    m = layers()
    rows, features, outputs = (310_000, 260, 260) if dtype == torch.bfloat16 else (
        160_000, 260, 260)
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, features, generator=gen, device="cuda").to(dtype)
    g = torch.randn(rows, outputs, generator=gen, device="cuda").to(dtype)
    w = torch.randn(outputs, features, generator=gen, device="cuda").to(dtype)
    b = torch.zeros(outputs, device="cuda", dtype=dtype)
    inputs = [t.requires_grad_() for t in (x, w, b)]
    dw, db = torch.autograd.grad(m.linear(*inputs), inputs[1:], g)
    held = m.dequantize(m.quantize(x.detach())).double()
    near(dw, (g.double().t() @ held).cpu(),
         ((rows + 2) * E * (g.double().abs().t() @ held.abs())).cpu(), dtype)
    near(db, g.double().sum(0).cpu(), ((rows + 2) * E * g.double().abs().sum(0)).cpu(), dtype)


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_linear_of_many_rows_of_whole_numbers(dtype):
    """The widest tiles of dW (they take dW's of 250 x 250 and these rows), odd
    shares of the rows: small whole numbers, whose sums float32 holds exactly;
    dW itself stays within what the type holds exactly."""
    m = layers()
    rows = 330_001 if dtype != torch.float32 else 170_001
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randint(-2, 3, (rows, 250), generator=gen, device="cuda").to(dtype)
    g = torch.zeros(rows, 250, device="cuda", dtype=dtype)
    at = torch.randint(0, rows, (20_000,), generator=gen, device="cuda")
    g[at, torch.arange(20_000, device="cuda") % 250] = 1
    w = torch.zeros(250, 250, device="cuda", dtype=dtype).requires_grad_()
    (dw,) = torch.autograd.grad(m.linear(x, w), w, g)
    want = (g.double().t() @ x.double())
    assert want.abs().max() <= 256  # exact in bfloat16's eight bits, too
    assert torch.equal(dw.double(), want)


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,features,outputs", [
    (90_001, 490, 500),   # several of the widest tiles of dW, ragged on both sides
    (310_000, 260, 260),  # narrow ones, as the widest would be mostly empty
    (20_001, 300, 900),   # as many shares of the rows as are no multiple of eight
    (3_001, 2_060, 2_070)])  # fewer shares than eight
def test_linear_of_many_dense_rows_of_whole_numbers(dtype, rows, features, outputs):
    """Every row counts: sums of small whole numbers stay below 2^24, which
    float32 holds exactly in any order, so each output is the exact sum,
    rounded once to the type. (A bound of n 2^-24 of the terms' sum would let
    a dW or db of zeros pass at these row counts.)"""
    m = layers()
    gen = torch.Generator(device="cuda").manual_seed(73)

    def whole(low, high, *shape):
        return torch.randint(low, high + 1, shape, generator=gen, device="cuda").to(dtype)

    x, g = whole(-2, 2, rows, features), whole(-1, 2, rows, outputs)
    w, b = whole(-1, 1, outputs, features), whole(-9, 9, outputs)
    inputs = [t.requires_grad_() for t in (x, w, b)]
    y = m.linear(*inputs)
    got = (y.detach(), *torch.autograd.grad(y, inputs, g))
    x, w, b, g = (t.detach().double() for t in (x, w, b, g))
    want = (x @ w.t() + b, g @ w, g.t() @ x, g.sum(0))
    for name, a, e in zip(("y", "dx", "dw", "db"), got, want):
        assert e.abs().max() < 2 ** 24 and torch.equal(a, e.to(dtype)), name


@gpu_test
def test_linear_of_a_matrix_larger_than_the_joining_grid():
    """More than 2^20 x 256 weights: the workgroups that join dW's partial
    sums take several stretches of it. Whole numbers: exact."""
    m = layers()
    rows, features, outputs = 9, 16384, 20001
    gen = generator(67)
    x = torch.randint(-9, 10, (rows, features), generator=gen).to(torch.bfloat16)
    g = torch.randint(-2, 3, (rows, outputs), generator=gen).to(torch.bfloat16)
    w = torch.zeros(outputs, features, dtype=torch.bfloat16, device="cuda").requires_grad_()
    b = torch.zeros(outputs, dtype=torch.bfloat16, device="cuda").requires_grad_()
    dw, db = torch.autograd.grad(m.linear(x.cuda(), w, b), (w, b), g.cuda())
    assert torch.equal(db.cpu().float(), g.float().sum(0))
    x, g = x.cuda().float(), g.cuda().float()
    for first in range(0, outputs, 4096):
        part = g[:, first:first + 4096]
        want = sum(part[r, :, None] * x[r, None, :] for r in range(rows))
        assert torch.equal(dw[first:first + 4096].float(), want), first


@gpu_test
def test_linear_gradients_asked_for_one_by_one():
    m = layers()
    x, w, b, g = (normal(*s, seed=i).cuda() for i, s in enumerate(((70, 48), (24, 48), (24,),
                                                                   (70, 24))))
    inputs = [t.clone().requires_grad_() for t in (x, w, b)]
    every = torch.autograd.grad(m.linear(*inputs), inputs, g)
    for i in range(3):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (one,) = torch.autograd.grad(m.linear(*some), some[i], g)
        assert torch.equal(one, every[i])
        (one,) = torch.autograd.grad(m.linear(*inputs), inputs[i], g)
        assert torch.equal(one, every[i])


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_whole_numbers_is_exact(dtype):
    """Small whole numbers: every product and sum is exact in float32, the
    kept rows are the rows, so all outputs equal the formula's, in any order
    of summation (and a wrong lane or a lost row shows)."""
    m = layers()
    gen = generator(9)
    x = torch.randint(-3, 4, (700, 200), generator=gen).to(dtype)
    w = torch.randint(-1, 2, (140, 200), generator=gen).to(dtype)
    g = torch.randint(-1, 2, (700, 140), generator=gen).to(dtype)
    inputs = [t.cuda().requires_grad_() for t in (x, w)]
    y = m.linear(*inputs)
    dx, dw = torch.autograd.grad(y, inputs, g.cuda())
    for got, want in ((y, x.double() @ w.double().t()), (dx, g.double() @ w.double()),
                      (dw, g.double().t() @ x.double())):
        assert torch.equal(got.cpu(), want.to(dtype))


@gpu_test
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_keeps_bad_values_to_their_place(dtype):
    m = layers()
    x, w, g = (normal(*s, seed=i, dtype=dtype) for i, s in enumerate(((200, 96), (40, 96),
                                                                       (200, 40))))
    x[150, 70] = math.inf
    inputs = [t.cuda().requires_grad_() for t in (x, w)]
    y = m.linear(*inputs)
    dx, dw = torch.autograd.grad(y, inputs, g.cuda())
    finite = torch.isfinite(y).all(1).cpu()
    assert not finite[150] and finite.sum() == 199
    assert torch.isfinite(dx).all()
    # The infinity's group of features, and no other.
    assert dw[:, 64:].isnan().all() and torch.isfinite(dw[:, :64]).all()


# --------------------------------------------------------------------------
# GPU: gradients against differences, and how the operators are called


def loss_of(name, x, w, b, g):
    if name == "layer_norm":
        return (oracle.layer_norm(x, w, b)[0] * g).sum()
    return (oracle.linear(x, w, b) * g).sum()


@gpu_test
@pytest.mark.parametrize("name", ["layer_norm", "linear"])
def test_gradients_against_differences(name):
    """Directional derivatives of the formulas by central differences in 64
    bits (step 1e-5: truncation and rounding both below 1e-8 relative),
    against float32 gradients of inputs that 8 bits keep without error, so
    the kept rows are the rows."""
    m = layers()
    gen = generator(17)
    x = torch.randint(-100, 101, (24, 64), generator=gen).float()
    x[:, ::32] = 100.0
    x[:, 1::32] = -100.0  # the middle of each row's range is 0
    outputs = 64 if name == "layer_norm" else 40
    w = normal(64, seed=1) if name == "layer_norm" else normal(40, 64, seed=1)
    b, g = normal(outputs, seed=2), normal(24, outputs, seed=3)
    inputs = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = m.layer_norm(*inputs, checkpoint="8bit") if name == "layer_norm" else m.linear(*inputs)
    grads = torch.autograd.grad(y, inputs, g.cuda())
    values = [t.double() for t in (x, w, b)]
    for i, grad in enumerate(grads):
        for seed in range(3):
            v = normal(*values[i].shape, seed=50 + seed).double()
            ends = []
            for sign in (1, -1):
                moved = list(values)
                moved[i] = values[i] + sign * 1e-5 * v
                ends.append(loss_of(name, *moved, g.double()))
            slope = ((ends[0] - ends[1]) / 2e-5).item()
            terms = grad.cpu().double() * v
            assert abs(terms.sum().item() - slope) <= 1e-5 * terms.abs().sum().item() + 1e-6


@gpu_test
@pytest.mark.parametrize("kind", ["sine", "gelu", "silu"])
def test_activation_gradient_against_differences(kind):
    m = layers()
    x, g = normal(20, 64, seed=1, scale=0.3), normal(20, 64, seed=2)
    on = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(m.activation(on, kind), on, g.cuda())
    z = oracle.kept(x)[2]
    ends = [oracle.activation(z + sign * 1e-6, kind, 30.0) for sign in (1, -1)]
    want = g.double() * (ends[0] - ends[1]) / 2e-6
    # Truncation: 30^3 1e-12 / 6; rounding: 1e-16 / 1e-6; float32: 30 16 E.
    assert (dx.cpu().double() - want).abs().max() <= 1e-4 * 30 * g.abs().max()


def every_operator(dtype=torch.bfloat16, rows=300, features=512):
    """Calls that give all outputs and gradients of each operator."""
    m = layers()
    x, g = normal(rows, features, seed=1, dtype=dtype), normal(rows, features, seed=2, dtype=dtype)
    w, b = normal(features, seed=3, dtype=dtype), normal(features, seed=4, dtype=dtype)
    big = normal(features, features, seed=5, dtype=dtype)
    x, g, w, b, big = (t.cuda() for t in (x, g, w, b, big))

    def train(call, *inputs):
        inputs = [t.detach().requires_grad_() for t in inputs]
        y = call(*inputs)
        return (y.detach(), *torch.autograd.grad(y, inputs, g))

    return {
        "checkpoint": lambda: (m.dequantize(m.quantize(x)),),
        "layer_norm": lambda: train(m.layer_norm, x, w, b),
        "layer_norm 8 bits": lambda: train(
            lambda *a: m.layer_norm(*a, checkpoint="8bit"), x, w, b),
        "sine": lambda: train(m.activation, x),
        "gelu": lambda: train(lambda z: m.activation(z, "gelu"), x),
        "linear": lambda: train(m.linear, x, big, b),
    }, (x, g, w, b, big)


@gpu_test
def test_results_repeat_bit_for_bit_on_any_stream():
    calls, _ = every_operator()
    first = {name: call() for name, call in calls.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = {name: call() for name, call in calls.items()}
    stream.synchronize()
    for name in first:
        for a, b in zip(first[name], second[name]):
            assert torch.equal(a, b), name


@gpu_test
def test_operators_in_a_graph():
    """Captured forward and backward passes replay with new inputs: each
    replay equals the eager result, with eager work between."""
    calls, inputs = every_operator()
    for name, call in calls.items():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = call()
        for seed in range(3):
            for i, t in enumerate(inputs):
                t.copy_(normal(*t.shape, seed=100 * seed + i, dtype=t.dtype))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outputs]
            for a, b in zip(got, call()):
                assert torch.equal(a, b), (name, seed)


@gpu_test
def test_expanded_and_strided_gradients():
    m = layers()
    x = normal(50, 96, seed=1).cuda()
    w, b = normal(96, seed=2).cuda(), normal(96, seed=3).cuda()
    big = normal(40, 96, seed=4).cuda()
    for call, outputs in ((lambda t: m.layer_norm(t, w, b, checkpoint="8bit"), 96),
                          (m.activation, 96), (lambda t: m.linear(t, big), 40)):
        scalar = torch.full((1, 1), 0.5).cuda()
        wide = normal(50, 3 * outputs, seed=5).cuda()
        for g in (scalar.expand(50, outputs), wide[:, outputs:2 * outputs],
                  normal(outputs, 50, seed=6).cuda().t()):
            results = []
            for grad in (g, g.contiguous()):
                on = x.clone().requires_grad_()
                results.append(torch.autograd.grad(call(on), on, grad)[0])
            assert torch.equal(*results)


@gpu_test
def test_strided_inputs_and_weights():
    m = layers()
    base = normal(60, 300, seed=1).cuda()
    w = normal(96, 40, seed=2).cuda().t()  # a transposed weight
    for x in (base[:, 10:106], base[::2, 8:104], base.view(3, 20, 300)[:, 2:9, :96]):
        for call in (lambda t: m.linear(t, w), m.activation, m.layer_norm,
                     lambda t: m.layer_norm(t, checkpoint="8bit")):
            results = []
            for t in (x, x.contiguous()):
                on = t.detach().requires_grad_()
                y = call(on)
                results.append((y, *torch.autograd.grad(y, on, torch.ones_like(y))))
            for a, b in zip(*results):
                assert torch.equal(a, b)


@gpu_test
def test_lazily_negated_views():
    """A view whose values are the negatives of what its memory holds (the
    imaginary part of a conjugate) is read as its values."""
    m = layers()
    x, g = normal(30, 64, seed=1).cuda(), normal(30, 64, seed=2).cuda()
    w, b, big = (normal(*s, seed=3).cuda() for s in ((64,), (64,), (64, 64)))
    pairs = [(torch.imag(torch.complex(t, t).conj()), -t) for t in (x[:, :1], x[0])]
    pairs += [(torch._neg_view(t), -t) for t in (x, g, w, b, big)]
    for lazy, plain in pairs:
        assert lazy.is_neg() and torch.equal(lazy, plain)
        a, e = m.quantize(lazy), m.quantize(plain)
        assert torch.equal(a.values, e.values) and torch.equal(a.exponents, e.exponents)
    _, (nx, px), (ng, pg), (nw, pw), (nb, pb), (nbig, pbig) = pairs[1:]
    for call, lazy, plain in (
            (m.activation, (nx,), (px,)),
            (m.layer_norm, (nx, nw, nb), (px, pw, pb)),
            (lambda *a: m.layer_norm(*a, checkpoint="8bit"), (nx, nw, nb), (px, pw, pb)),
            (m.linear, (nx, nbig, nb), (px, pbig, pb))):
        results = []
        for inputs, grad in ((lazy, ng), (plain, pg)):
            inputs = [t.detach().requires_grad_() for t in inputs]
            y = call(*inputs)
            results.append((y, *torch.autograd.grad(y, inputs, grad)))
        for a, e in zip(*results):
            assert torch.equal(a, e)


@gpu_test
def test_shared_and_broadcast_inputs():
    """An input used twice and a weight expanded from fewer values: autograd
    adds what the operators return."""
    m = layers()
    x, w = normal(30, 64, seed=1).cuda(), normal(64, 64, seed=2).cuda()
    on = x.clone().requires_grad_()
    y = m.linear(m.layer_norm(on), w) + m.layer_norm(on)
    (both,) = torch.autograd.grad(y, on, torch.ones_like(y))
    on1, on2 = x.clone().requires_grad_(), x.clone().requires_grad_()
    y = m.linear(m.layer_norm(on1), w) + m.layer_norm(on2)
    one, two = torch.autograd.grad(y, (on1, on2), torch.ones_like(y))
    torch.testing.assert_close(both, one + two, atol=1e-5, rtol=1e-5)
    scale = torch.tensor([1.5]).cuda().requires_grad_()
    y = m.layer_norm(x, scale.expand(64))
    (g,) = torch.autograd.grad(y.square().sum(), scale)
    h = m.layer_norm(x)
    torch.testing.assert_close(g[0], (2 * 1.5 * h.square()).sum(), atol=1e-2, rtol=1e-5)


@gpu_test
def test_no_rows():
    m = layers()
    for dtype in DTYPES:
        x = torch.zeros(0, 48, dtype=dtype).cuda().requires_grad_()
        w = torch.ones(48, dtype=dtype).cuda().requires_grad_()
        big = torch.ones(20, 48, dtype=dtype).cuda().requires_grad_()
        b = torch.ones(20, dtype=dtype).cuda().requires_grad_()
        assert m.dequantize(m.quantize(x.detach())).shape == (0, 48)
        y = m.activation(x)
        assert torch.autograd.grad(y, x, torch.zeros_like(y))[0].shape == (0, 48)
        y = m.layer_norm(x, w, w.detach(), checkpoint="8bit")
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert dx.shape == (0, 48) and torch.equal(dw, torch.zeros_like(dw))
        y = m.linear(x, big, b)
        dx, dw, db = torch.autograd.grad(y, (x, big, b), torch.zeros_like(y))
        assert y.shape == (0, 20) and dx.shape == (0, 48)
        assert torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, torch.zeros_like(db))


@gpu_test
def test_second_derivatives_are_refused():
    m = layers()
    x = normal(4, 32, seed=1).cuda().requires_grad_()
    w = normal(8, 32, seed=2).cuda().requires_grad_()
    for call in (m.layer_norm, m.activation, lambda t: m.linear(t, w)):
        y = call(x)
        (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            dx.sum().backward()


@gpu_test
def test_forward_mode_and_tracing_are_refused_on_the_device():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x = normal(2, 8, seed=1).cuda()
    calls = layer_calls("cuda")
    refuses_what_would_lose_a_result(calls, x)
    for name, call in calls.items():
        on = x.clone().requires_grad_()
        y = call(on)
        g = torch.ones_like(y)

        def back(t):
            return torch.autograd.grad(y, on, t, retain_graph=True)[0]

        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            make_fx(back)(g)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode"):
            back(forward_ad.make_dual(g, torch.ones_like(g)))
        for transform in (torch.func.vmap, torch.func.functionalize,
                          lambda f: lambda t: torch.func.jvp(f, (t,), (t,))):
            with pytest.raises(RuntimeError):
                transform(call)(x)
        with pytest.raises(RuntimeError), FakeTensorMode(allow_non_fake_inputs=True) as mode:
            call(mode.from_tensor(x))
        # None of it stays behind.
        assert torch.equal(call(x), y.detach())
        assert torch.isfinite(back(g)).all()


@gpu_test
def test_refusals():
    m = layers()
    x = torch.zeros(4, 32, device="cuda")
    bf = x.bfloat16()
    cases = [
        (lambda: m.quantize(x.double()), "float32, bfloat16 or float16"),
        (lambda: m.quantize(x.int()), "float32, bfloat16 or float16"),
        (lambda: m.quantize(x[:, :0]), "at least one feature"),
        (lambda: m.quantize(torch.zeros((), device="cuda")), "at least one feature"),
        (lambda: m.dequantize(m.Checkpoint(x.char(), x[:, :1].byte(), (4, 33), x.dtype)),
         "do not hold a checkpoint"),
        (lambda: m.dequantize(m.quantize(x), torch.int32), "reads back as"),
        (lambda: m.layer_norm(x, torch.zeros(31, device="cuda")), r"shape \(32,\)"),
        (lambda: m.layer_norm(x, torch.zeros(32)), "device of x"),
        (lambda: m.layer_norm(x, torch.zeros(32, device="cuda").half()), "type of x or float32"),
        (lambda: m.layer_norm(bf, torch.zeros(32, device="cuda"),
                              torch.zeros(32, device="cuda").bfloat16()), "one type"),
        (lambda: m.linear(x, torch.zeros(8, 31, device="cuda")), r"shape \(8, 32\)"),
        (lambda: m.linear(x, torch.zeros(32, device="cuda")), r"\(outputs, features\)"),
        (lambda: m.linear(bf, torch.zeros(8, 32, device="cuda")), "type of x"),
        (lambda: m.linear(x, torch.zeros(8, 32, device="cuda"), torch.zeros(9, device="cuda")),
         r"shape \(8,\)"),
    ]
    for call, text in cases:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(RuntimeError, match="at most 16384"):
        m.layer_norm(torch.zeros(2, 16385, device="cuda"))


@gpu_test
def test_offsets_past_32_bits():
    """Rows whose offsets pass 2^31 values: the last ones are what they are
    when they are alone."""
    m = layers()
    rows, features = (1 << 31) // 256 + 77, 256
    gen = torch.Generator(device="cuda").manual_seed(1)
    tail = torch.randn(300, features, generator=gen, device="cuda").bfloat16()
    x = torch.zeros(rows, features, device="cuda", dtype=torch.bfloat16)
    x[-300:] = tail
    kept, alone = m.quantize(x), m.quantize(tail)
    assert torch.equal(kept.values[-300:], alone.values)
    assert torch.equal(kept.exponents[-300:], alone.exponents)
    assert torch.equal(m.dequantize(kept)[-300:], m.dequantize(alone))
    del kept
    w = torch.randn(64, features, generator=gen, device="cuda").bfloat16() / 16
    g = torch.zeros(rows, 64, device="cuda", dtype=torch.bfloat16)
    g[-300:] = torch.randn(300, 64, generator=gen, device="cuda").bfloat16()
    for call, grad in ((lambda t, v: m.linear(t, v), g),
                       (lambda t, v: m.layer_norm(t, v[0], checkpoint="8bit"), None),
                       (lambda t, v: m.activation(t), None)):
        results = []
        for t in (x, tail):
            on, v = t.detach().requires_grad_(), w.detach().requires_grad_()
            y = call(on, v)
            dy = (grad[-len(t):] if grad is not None else
                  torch.zeros_like(t).index_copy_(0, torch.arange(len(t) - 300, len(t),
                                                                  device="cuda"), tail))
            dx, dv = torch.autograd.grad(y, (on, v), dy, allow_unused=True)
            results.append((y[-300:].detach().clone(), dx[-300:].clone(), dv))
            del y, dx, dy, on
        (y1, dx1, dw1), (y2, dx2, dw2) = results
        assert torch.equal(y1, y2) and torch.equal(dx1, dx2)
        if dw1 is not None:
            # The same few terms, summed in another order: one unit in
            # bfloat16's last place.
            assert (dw1.float() - dw2.float()).abs().max() <= 2.0 ** -7 * dw2.float().abs().max()


@gpu_test
def test_more_rows_than_one_launch_takes():
    """A row of one feature takes four chunks, a thread four chunks: 2^32 rows
    would be 2^32 threads, more than a launch takes, and 2^30 rows are as many
    as one is given. A pattern of odd length repeats over the rows, and so do
    the results."""
    m = layers()
    torch.cuda.empty_cache()
    period = 1_000_003
    base = normal(period, seed=71, dtype=torch.bfloat16).cuda()[:, None]

    def repeats(got, want, times):
        assert torch.equal(got.reshape(times, -1), want.reshape(1, -1).expand(times, -1))

    times = (1 << 32) // period + 2
    repeats(m.activation(base.repeat(times, 1), "silu"), m.activation(base, "silu"), times)
    torch.cuda.empty_cache()
    times = (1 << 30) // period + 2
    results = []
    for x in (base, base.repeat(times, 1)):
        on = x.requires_grad_()
        y = m.activation(on, "silu")
        (dx,) = torch.autograd.grad(y, on, x.detach())
        kept = m.quantize(x)
        results.append((y.detach(), dx, kept.values, kept.exponents, m.dequantize(kept)))
        del on, y, dx, kept, x
    for want, got in zip(*results):
        repeats(got, want, times)
    del results, got
    torch.cuda.empty_cache()


@gpu_test
def test_linear_of_as_many_tiles_as_a_launch_takes():
    """2^34 weights are 2^20 tiles of dW; eight workgroups of 512 threads to
    each would be 2^32 threads. Whole numbers: exact."""
    m = layers()
    torch.cuda.empty_cache()
    rows, side = 9, 1 << 17
    gen = torch.Generator(device="cuda").manual_seed(72)
    x = torch.randint(-9, 10, (rows, side), generator=gen, device="cuda").to(torch.bfloat16)
    g = torch.randint(-2, 3, (rows, side), generator=gen, device="cuda").to(torch.bfloat16)
    w = torch.zeros(side, side, dtype=torch.bfloat16, device="cuda").requires_grad_()
    (dw,) = torch.autograd.grad(m.linear(x, w), w, g)
    x, g = x.float(), g.float()
    for first in range(0, side, 2048):
        want = g[:, first:first + 2048].t() @ x
        assert torch.equal(dw[first:first + 2048].float(), want), first
    del w, dw, want
    torch.cuda.empty_cache()
