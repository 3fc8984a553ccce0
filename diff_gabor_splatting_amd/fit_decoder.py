"""Fit a stripe texture through a decoder: latents -> layers -> neural surfels -> renderer.

A flat grid of surfels three units in front of the 32 x 32 camera of
``fit_texture``, each with a learned latent vector. A decoder shared by all
of them (layer norm, linear, sine, linear: ``layers``) turns a latent into the
57 values of its SIREN, which the neural renderer composites; Adam (lr 0.001)
fits latents and decoder together to the stripes 0.5 + 0.4 cos(0.7 x) masked
by the rendered alpha. The layers keep their inputs in 8 bits for the backward
pass (``--checkpoint full`` keeps the layer norm's whole).

Initial parameters are drawn on the CPU from a seeded generator, and both the
layers and the renderer can be replaced (the tests run the same problem
through plain 64-bit operations and the oracle's renderer).

    python -m diff_gabor_splatting_amd.fit_decoder --steps 100 --dtype bfloat16
"""

from __future__ import annotations

import argparse
import math

import torch

from .fit_texture import SIZE

NEURAL_SHAPES = {"input_weights": (6, 5), "input_biases": (6,), "output_weights": (3, 6),
                 "output_biases": (3,)}
OUTPUTS = sum(math.prod(shape) for shape in NEURAL_SHAPES.values())  # 57
OMEGA = 30.0


def decoder_problem(side: int = 8, features: int = 64, hidden: int = 96, device="cuda",
                    dtype=torch.float32, decoder_dtype=None, seed: int = 3):
    """(fixed renderer inputs, fitted parameters, target stripes [1, H, W, 3])
    of a side x side grid of surfels."""
    gen = torch.Generator().manual_seed(seed)
    decoder_dtype = decoder_dtype or dtype
    n = side * side

    def uniform(*shape, bound):
        return ((torch.rand(shape, generator=gen, dtype=torch.float64) * 2 - 1) * bound)

    at = (torch.arange(side, dtype=torch.float64) + 0.5) / side * 2 - 1
    y, x = torch.meshgrid(at, at, indexing="ij")
    means = torch.stack((x.reshape(-1) * 0.8, y.reshape(-1) * 0.8, torch.full((n,), 3.0)), 1)
    fixed = {
        "means": means,
        "quaternions": torch.tensor([[1.0, 0.0, 0.0, 0.0]]).expand(n, 4),
        "scales": torch.full((n, 2), 0.8 / side),
        "opacities": torch.full((n,), 0.8),
        "view_matrices": torch.eye(4)[None],
        "intrinsics": torch.tensor([[[40.0, 0.0, 15.5], [0.0, 40.0, 15.5], [0.0, 0.0, 1.0]]]),
    }
    fixed = {k: v.to(dtype).to(device).contiguous() for k, v in fixed.items()}
    # The head starts from the texture fit's SIREN (input weights within 1/5,
    # output weights within 1/30), which the latents then vary.
    head_bias = torch.cat((uniform(30, bound=1 / 5), torch.zeros(6, dtype=torch.float64),
                           uniform(18, bound=1 / 30), torch.zeros(3, dtype=torch.float64)))
    fitted = {
        "latents": uniform(n, features, bound=1.0),
        "norm_weight": torch.ones(features),
        "norm_bias": torch.zeros(features),
        "hidden_weight": uniform(hidden, features, bound=math.sqrt(6 / features) / OMEGA),
        "hidden_bias": uniform(hidden, bound=1 / OMEGA),
        "head_weight": uniform(OUTPUTS, hidden, bound=0.1 / math.sqrt(hidden)),
        "head_bias": head_bias,
    }
    fitted = {k: v.to(decoder_dtype).to(device).requires_grad_() for k, v in fitted.items()}
    stripes = 0.5 + 0.4 * torch.cos(0.7 * torch.arange(SIZE, dtype=dtype, device=device))
    return fixed, fitted, stripes[None, None, :, None].expand(1, SIZE, SIZE, 3).contiguous()


def decode(fitted: dict, layers, checkpoint: str = "8bit") -> dict:
    """The neural renderer's appearance inputs of every surfel, in float32 (or
    in float64 where the decoder works in it)."""
    h = layers.layer_norm(fitted["latents"], fitted["norm_weight"], fitted["norm_bias"],
                          checkpoint=checkpoint)
    h = layers.linear(h, fitted["hidden_weight"], fitted["hidden_bias"])
    h = layers.activation(h, "sine", OMEGA)
    h = layers.linear(h, fitted["head_weight"], fitted["head_bias"])
    if h.dtype != torch.float64:
        h = h.float()
    parts = h.split([math.prod(shape) for shape in NEURAL_SHAPES.values()], 1)
    return {name: part.reshape(-1, *shape).contiguous()
            for (name, shape), part in zip(NEURAL_SHAPES.items(), parts)}


def fit_decoder(steps: int, device="cuda", dtype=torch.float32, decoder_dtype=None, layers=None,
                render=None, checkpoint: str = "8bit", verbose: bool = False, **problem) -> dict:
    """Run the fit; returns the losses and the final render [H, W, 3]."""
    if layers is None:
        from . import layers
    if render is None:
        from .rendering import rasterize_neural_gabors as render
    fixed, fitted, target = decoder_problem(device=device, dtype=dtype,
                                            decoder_dtype=decoder_dtype, **problem)
    optimizer = torch.optim.Adam(list(fitted.values()), lr=0.001)
    losses = []
    for step in range(steps):
        optimizer.zero_grad(set_to_none=True)
        rgb, alpha, _ = render(**fixed, **decode(fitted, layers, checkpoint), width=SIZE,
                               height=SIZE)
        loss = (rgb - target * alpha.detach()).square().mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if verbose and (step == 0 or step == steps - 1):
            print(f"step={step + 1} loss={losses[-1]:.6f}", flush=True)
    if not all(math.isfinite(value) for value in losses):
        raise RuntimeError("optimization produced non-finite losses")
    with torch.no_grad():
        rgb, _, _ = render(**fixed, **decode(fitted, layers, checkpoint), width=SIZE,
                           height=SIZE)
    return {"losses": losses, "final": rgb[0].cpu()}


def main(argv=None) -> dict:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--side", type=int, default=8, help="surfels along each side of the grid")
    parser.add_argument("--features", type=int, default=64)
    parser.add_argument("--hidden", type=int, default=96)
    parser.add_argument("--dtype", choices=["float32", "bfloat16", "float16"],
                        default="float32", help="of the latents and the decoder")
    parser.add_argument("--checkpoint", choices=["full", "8bit"], default="8bit",
                        help="what the layer norm keeps")
    args = parser.parse_args(argv)
    if min(args.steps, args.side, args.features, args.hidden) < 1:
        parser.error("--steps, --side, --features and --hidden must be positive")
    return fit_decoder(args.steps, decoder_dtype=getattr(torch, args.dtype), side=args.side,
                       features=args.features, hidden=args.hidden, checkpoint=args.checkpoint,
                       verbose=True)


if __name__ == "__main__":
    main()
