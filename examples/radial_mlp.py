"""Train a radial MLP of the non-linear interaction block's form on the pair distances of molecules.

    PYTHONPATH=. python examples/radial_mlp.py [--structures 32] [--steps 200] [--max-norm 10]

Each hidden layer is Linear -> LayerNorm -> SiLU, the last one plain.  The
framework's neighbour list gives the edges; the MLP maps eight Bessel functions
of an edge's length to weights per channel, here fitted to those of a second MLP
of the same form, so the loss can go to zero.  The layer norm with its SiLU and
the clipping of the gradients are the framework's operators; the hidden layers'
gradients at their gains and biases are sums over all edges.
"""

from __future__ import annotations

import argparse
import math

import numpy as np
import torch

from mace_mlx_b200 import norms
from mace_mlx_b200.model import MACEModel
from mace_mlx_b200.spec import ModelSpec
from mace_mlx_b200.structures import molecule_batch
from mace_mlx_b200.weights import random_config, random_weights


def edge_features(n_structures: int, seed: int = 0, device: int = 0, num_bessel: int = 8) -> torch.Tensor:
    """Bessel functions of the length of every edge within 5 A of a batch of molecules (E, num_bessel)."""
    config = random_config("small", z_table=[1, 6, 7, 8], r_max=5.0, avg_num_neighbors=12.0)
    model = MACEModel(config=config, weights=random_weights(ModelSpec.from_config(config), seed), device=device)
    st = molecule_batch(n_structures, seed)
    ptr = torch.as_tensor(np.searchsorted(st.batch, np.arange(n_structures + 1)).astype(np.int32), device=model.device)
    pos = torch.tensor(st.positions, dtype=torch.float64, device=model.device)
    edges = model.neighbour_list(pos, None, st.pbc, ptr, model.r_max)
    i, j = edges.sender[:edges.n_edges].long(), edges.receiver[:edges.n_edges].long()
    r = (pos[j] - pos[i]).norm(dim=1, keepdim=True)
    n = torch.arange(1, num_bessel + 1, dtype=torch.float64, device=model.device)
    return (math.sqrt(2.0 / model.r_max) * torch.sin(n * math.pi * r / model.r_max) / r).float()


class RadialMLP(torch.nn.Module):
    def __init__(self, widths: list[int], generator: torch.Generator):
        super().__init__()

        def parameter(*shape, scale=1.0, offset=0.0):
            values = torch.randn(*shape, generator=generator, device=generator.device)
            return torch.nn.Parameter(offset + scale * values)

        pairs = list(zip(widths, widths[1:]))
        self.weights = torch.nn.ParameterList(parameter(m, k, scale=k**-0.5) for k, m in pairs)
        self.biases = torch.nn.ParameterList(parameter(m, scale=0.1) for _, m in pairs)
        self.gains = torch.nn.ParameterList(parameter(m, scale=0.1, offset=1.0) for _, m in pairs[:-1])
        self.shifts = torch.nn.ParameterList(parameter(m, scale=0.1) for _, m in pairs[:-1])

    def forward(self, x):
        for i, (weight, bias) in enumerate(zip(self.weights, self.biases)):
            x = torch.nn.functional.linear(x, weight, bias)
            if i < len(self.gains):
                x = norms.layer_norm(x, self.gains[i], self.shifts[i], activation="silu")
        return x


def train(n_structures: int = 32, steps: int = 200, channels: int = 128, seed: int = 0, lr: float = 1e-2,
          max_norm: float = 10.0) -> tuple[list[float], list[float]]:
    """Fits the MLP; the loss (mean squared error) and the gradients' norm at every step."""
    x = edge_features(n_structures, seed)
    generator = torch.Generator(x.device).manual_seed(seed)
    widths = [x.shape[1], 64, 64, 64, channels]
    with torch.no_grad():
        target = RadialMLP(widths, generator)(x)
    mlp = RadialMLP(widths, generator)
    optimiser = torch.optim.Adam(mlp.parameters(), lr=lr)
    losses, sizes = [], []
    for _ in range(steps):
        optimiser.zero_grad(set_to_none=True)
        loss = (mlp(x) - target).square().mean()
        loss.backward()
        sizes.append(norms.clip_grads([p.grad for p in mlp.parameters()], max_norm))
        optimiser.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), torch.stack(sizes).tolist()


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--structures", type=int, default=32)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--max-norm", type=float, default=10.0)
    args = parser.parse_args()
    losses, sizes = train(args.structures, args.steps, max_norm=args.max_norm)
    every = max(1, len(losses) // 10)
    for step in [*range(0, len(losses) - 1, every), len(losses) - 1]:
        print(f"step {step:4d}  loss {losses[step]:.4e}  gradient norm {sizes[step]:.3e}")


if __name__ == "__main__":
    main()
