"""The decoder's layers and the renderer in one training loop (fit_decoder).

The problem itself is pinned on the CPU: through plain 64-bit operations
(layers kept whole) and the oracle's renderer the loss must fall. The HIP
path must follow it: at the first step to the rounding of float32 (the
forward pass does not depend on what is kept), and to a loss as low at the end.
"""

import types

import pytest
import torch

from diff_gabor_splatting_amd.fit_decoder import (OUTPUTS, decode, decoder_problem, fit_decoder,
                                                  main)
from oracle import render as oracle_render

STEPS = 25

plain_layers = types.SimpleNamespace(
    layer_norm=lambda x, w, b, checkpoint: torch.nn.functional.layer_norm(x, x.shape[-1:], w, b),
    linear=torch.nn.functional.linear,
    activation=lambda x, kind, omega: torch.sin(omega * x),
)


def oracle_renderer(**arguments):
    maps, meta, _ = oracle_render.rasterize_neural_gabors(**arguments)
    return maps[..., :3], maps[..., 3:4], meta


_PLAIN = {}


def plain_fit():
    if not _PLAIN:
        _PLAIN.update(fit_decoder(STEPS, device="cpu", dtype=torch.float64, layers=plain_layers,
                                  render=oracle_renderer, side=4, features=32, hidden=40))
    return _PLAIN


def test_plain_fit_reduces_the_loss():
    losses = plain_fit()["losses"]
    assert losses[-1] < 0.5 * losses[0]


def test_decoded_shapes():
    _, fitted, target = decoder_problem(side=2, features=16, hidden=24, device="cpu",
                                        dtype=torch.float64)
    out = decode(fitted, plain_layers)
    assert OUTPUTS == 57 and target.shape == (1, 32, 32, 3)
    assert [tuple(v.shape) for v in out.values()] == [(4, 6, 5), (4, 6), (4, 3, 6), (4, 3)]


def test_arguments():
    with pytest.raises(SystemExit):
        main(["--steps", "0"])


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("dtype,first", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("checkpoint", ["8bit", "full"])
def test_hip_fit_follows_the_plain_one(dtype, first, checkpoint):
    """First loss: the maps agree to 1e-5 in float32; in bfloat16 the decoded
    values are off by 2^-8 of their size. Last loss: gradients taken at 8-bit
    inputs are off by parts of a hundred, so the paths part, but they descend
    as the plain one does."""
    losses = fit_decoder(STEPS, decoder_dtype=dtype, checkpoint=checkpoint, side=4, features=32,
                         hidden=40)["losses"]
    plain = plain_fit()["losses"]
    assert abs(losses[0] - plain[0]) <= first * plain[0]
    assert losses[-1] < 0.6 * losses[0]


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_kept_bytes():
    """What the decoder saves for its backward pass, beside its parameters and
    the layer norm's two statistics of a row: 33/32 of a byte for each input
    value of each layer."""
    from diff_gabor_splatting_amd import layers

    _, fitted, _ = decoder_problem(side=16, features=64, hidden=96, dtype=torch.float32)
    parameters = {v.data_ptr() for v in fitted.values()}
    sizes = {}

    def pack(t):
        if t.data_ptr() not in parameters:
            sizes[t.data_ptr()] = t.nbytes
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        h = layers.layer_norm(fitted["latents"], fitted["norm_weight"], fitted["norm_bias"],
                              checkpoint="8bit")
        h = layers.linear(h, fitted["hidden_weight"], fitted["hidden_bias"])
        h = layers.activation(h, "sine")
        layers.linear(h, fitted["head_weight"], fitted["head_bias"])
    rows = 256
    inputs = 64 + 64 + 96 + 96
    assert sum(sizes.values()) == rows * (inputs + inputs // 32 + 2 * 4)
