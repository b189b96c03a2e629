"""A small model of atoms out of the operators of the block, trained on synthetic energies:

* `embedding_lookup`: a row of a table for each atom, by its species;
* `grouped_matrix_product`: linear maps whose matrices depend on the species (experts, for tokens);
* `gated_residual_norm`: what a layer computed is normed, gated and added to the stream, which is normed for the next layer.

Atoms are sorted by species once per batch (`mops_b200.sort_indices`), so that those of a species are neighbours.

    python examples/species_blocks.py [--steps 100] [--dtype float32]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import mops_b200  # noqa: E402
import mops_b200.torch as mt  # noqa: E402


class Layer(torch.nn.Module):
    def __init__(self, species, channels, hidden):
        super().__init__()
        self.widen = torch.nn.Parameter(torch.randn(species, channels, hidden) * channels ** -0.5)
        self.narrow = torch.nn.Parameter(torch.randn(species, hidden, channels) * hidden ** -0.5)
        self.gate = torch.nn.Parameter(torch.zeros(species, channels, 1))
        self.scale = torch.nn.Parameter(torch.full((channels,), 0.5))
        self.weight_branch = torch.nn.Parameter(torch.ones(channels))
        self.weight_output = torch.nn.Parameter(torch.ones(channels))

    def forward(self, stream, normed, offsets):
        hidden = torch.nn.functional.silu(mt.grouped_matrix_product(normed, self.widen, offsets))
        branch = mt.grouped_matrix_product(hidden, self.narrow, offsets)
        gate = mt.grouped_matrix_product(normed, self.gate, offsets)
        return mt.gated_residual_norm(stream, branch, gate, self.scale, self.weight_branch, self.weight_output, 1e-5)


class Model(torch.nn.Module):
    def __init__(self, species=20, channels=128, hidden=256, layers=2):
        super().__init__()
        self.species = species
        self.table = torch.nn.Parameter(torch.randn(species, channels) * channels ** -0.5)
        self.layers = torch.nn.ModuleList(Layer(species, channels, hidden) for _ in range(layers))
        self.readout = torch.nn.Parameter(torch.zeros(channels))

    def forward(self, species, charges):
        """An energy for each atom. species: int32, in order (of `by_species`); charges: a number for each atom."""
        boundaries = torch.arange(self.species + 1, device=species.device, dtype=torch.int32)
        offsets = torch.searchsorted(species, boundaries, out_int32=True)
        stream = mt.embedding_lookup(self.table, species, math.sqrt(self.table.shape[1]))
        stream = stream * (1 + charges[:, None].to(stream.dtype))
        normed = stream
        for layer in self.layers:
            stream, normed = layer(stream, normed, offsets)
        return normed.float() @ self.readout.float()


def by_species(species, n_species, *others):
    """The atoms in the order of their species (those of one in the order they had)."""
    ordered, order = mops_b200.sort_indices(species, n_species)
    return (ordered, *(t[order.long()] for t in others))


def batch(model, structures, atoms, generator, device="cuda"):
    """Species, a charge for each atom, the structure it belongs to, and energies of the structures that depend on both."""
    n = structures * atoms
    species = torch.randint(model.species, (n,), generator=generator, device=device, dtype=torch.int32)
    charges = torch.randn(n, generator=generator, device=device) * 0.5
    structure = torch.arange(n, device=device) // atoms
    energies = torch.zeros(structures, device=device).index_add_(0, structure, torch.sin(species.float()) * (1 + charges))
    return (*by_species(species, model.species, charges, structure), energies)


def train(steps=100, structures=64, atoms=100, dtype=torch.bfloat16, seed=0, **sizes):
    """Trains a new model; returns it with the losses."""
    torch.manual_seed(seed)
    generator = torch.Generator(device="cuda").manual_seed(seed)
    model = Model(**sizes).to(device="cuda", dtype=dtype)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        species, charges, structure, energies = batch(model, structures, atoms, generator)
        of_atoms = model(species, charges)
        predicted = torch.zeros_like(energies).index_add_(0, structure, of_atoms)
        loss = torch.mean((predicted - energies) ** 2) / atoms
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return model, torch.stack(losses).tolist()


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float16", "float32", "float64"])
    arguments = parser.parse_args()
    model, losses = train(arguments.steps, dtype=getattr(torch, arguments.dtype))
    for step in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {step:4d}  loss {losses[step]:.4f}")
    print(f"last step  loss {losses[-1]:.4f}")
    with torch.no_grad():  # one atom at a time, as it would be asked for
        energy = model(torch.tensor([3], device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda"))
    print(f"an atom of species 3: {energy.item():.4f} (the data's: {math.sin(3):.4f})")


if __name__ == "__main__":
    main()
