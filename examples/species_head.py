"""Train a species-dependent energy head on the node features of a frozen MACE model.

    PYTHONPATH=. python examples/species_head.py [--structures 32] [--steps 200] [--max-norm 10]

The model's own step (``MACEModel.evaluate``) gives the features h (N, d, C) of
its first layer: a scalar and a vector per channel.  The head is the pair of
species-indexed parts that MACE's layers have,

    y[n]    = h[n] W[z_n] / sqrt(C)  (+ table[z_n] on the scalars)
    E_graph = sum over its atoms of  sum_c a_c tanh(y0_c) + b_c |y1_c|^2

trained with the species operators: atoms are grouped by species once, the map
keeps h for the weight gradient in 8 bits, and the backward gives the gradients
of the matrices and of the table.  The energies to fit are those of a second
head of the same form, so the loss can go to zero.
"""

from __future__ import annotations

import argparse

import numpy as np
import torch

from mace_mlx_b200 import norms
from mace_mlx_b200 import species as sp
from mace_mlx_b200.model import MACEModel
from mace_mlx_b200.spec import ModelSpec
from mace_mlx_b200.structures import molecule_batch
from mace_mlx_b200.weights import random_config, random_weights


def frozen_features(n_structures: int, seed: int = 0, device: int = 0):
    """(h (N, 4, C), species (N,) int32, graph of each atom (N,)) of a batch of molecules under a random-init model."""
    config = random_config("medium", z_table=[1, 6, 7, 8], r_max=5.0, avg_num_neighbors=12.0)
    model = MACEModel(config=config, weights=random_weights(ModelSpec.from_config(config), seed), device=device)
    st = molecule_batch(n_structures, seed)
    graph = torch.as_tensor(st.batch, dtype=torch.int64, device=model.device)
    ptr = torch.as_tensor(np.searchsorted(st.batch, np.arange(n_structures + 1)).astype(np.int32), device=model.device)
    pos = torch.tensor(st.positions, dtype=torch.float64, device=model.device)
    species = torch.as_tensor(model.species_index(st.numbers), dtype=torch.int32, device=model.device)
    edges = model.neighbour_list(pos, None, st.pbc, ptr, model.r_max)
    model.evaluate(pos.float(), None, species, ptr, edges, forces=False)
    h = model.debug_buffer("h_out", 0).reshape(len(st), 4, -1)
    return h / h.square().mean().sqrt(), species, graph


class SpeciesHead(torch.nn.Module):
    def __init__(self, num_elements: int, channels: int, width: int, generator: torch.Generator):
        super().__init__()

        def parameter(*shape):
            return torch.nn.Parameter(torch.randn(*shape, generator=generator, device=generator.device))

        self.weight = parameter(num_elements, channels, width)
        self.table = parameter(num_elements, width)
        self.scalar, self.vector = parameter(width), parameter(width)
        self.alpha = channels**-0.5

    def forward(self, h, species, groups, graph, n_graphs: int):
        y = sp.species_linear(h, self.weight, groups, alpha=self.alpha, checkpoint=True)
        y0 = y[:, 0] + sp.species_embedding(self.table, species, groups=groups)
        atom = torch.tanh(y0) @ self.scalar + y[:, 1:].square().sum(1) @ self.vector
        return torch.zeros(n_graphs, device=h.device).index_add(0, graph, atom) / graph.bincount(minlength=n_graphs)


def train(n_structures: int = 32, steps: int = 200, width: int = 64, seed: int = 0, lr: float = 2e-2,
          max_norm: float | None = None) -> list[float]:
    """Fits the head, its gradients clipped to ``max_norm`` where one is given; the loss (mean squared error of the
    energies per atom) at every step."""
    h, species, graph = frozen_features(n_structures, seed)
    groups = sp.group_species(species, 4)
    generator = torch.Generator(h.device).manual_seed(seed)
    target = SpeciesHead(4, h.shape[2], width, generator)
    with torch.no_grad():
        energy = target(h, species, groups, graph, n_structures)
    head = SpeciesHead(4, h.shape[2], width, generator)
    optimiser = torch.optim.Adam(head.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        optimiser.zero_grad(set_to_none=True)
        loss = (head(h, species, groups, graph, n_structures) - energy).square().mean()
        loss.backward()
        if max_norm is not None:
            norms.clip_grads([p.grad for p in head.parameters()], max_norm)
        optimiser.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--structures", type=int, default=32)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--max-norm", type=float, default=None, help="bound of the gradients' norm (none)")
    args = parser.parse_args()
    losses = train(args.structures, args.steps, max_norm=args.max_norm)
    for step in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {step:4d}  loss {losses[step]:.4e}")
    print(f"step {len(losses) - 1:4d}  loss {losses[-1]:.4e}")


if __name__ == "__main__":
    main()
