"""A model that guesses the species of masked atoms (or masked words), out of the operators of the block and those that a training step has
behind them: species are looked up in a table, every layer is a gated feed-forward layer with weights for each environment
(``grouped_gated_product`` and the product back), joined to the stream by ``gated_residual_norm``, and the answer is the softmax over the same
table's rows: ``linear_cross_entropy`` takes the loss of the masked atoms without their logits. Gradients are clipped together.

    python examples/masked_species.py [--atoms 4096] [--steps 300] [--dtype bf16]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import mops_b200.torch as mt  # noqa: E402

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


class MaskedSpecies(torch.nn.Module):
    def __init__(self, species, environments, channels, width, layers, dtype, seed=0):
        super().__init__()
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(*shape):
            return torch.nn.Parameter((torch.randn(shape, generator=gen, device="cuda") * shape[-2] ** -0.5).to(dtype))

        vector = lambda value: torch.nn.Parameter(torch.full((channels,), value, device="cuda", dtype=dtype))
        self.table = torch.nn.Parameter((torch.randn((species, channels), generator=gen, device="cuda") * channels ** -0.5).to(dtype))
        self.inner = torch.nn.ParameterList([matrix(environments, channels, 2 * width) for _ in range(layers)])
        self.outer = torch.nn.ParameterList([matrix(environments, width, channels) for _ in range(layers)])
        self.vectors = torch.nn.ParameterList([torch.nn.ParameterList([vector(0.5), vector(1.0), vector(1.0)]) for _ in range(layers)])

    def forward(self, species, offsets):
        """Rows in front of the table, for atoms sorted by environment (``offsets``)."""
        stream = mt.embedding_lookup(self.table, species, math.sqrt(self.table.shape[1]))
        normed = stream
        for inner, outer, (scale, weight_branch, weight_output) in zip(self.inner, self.outer, self.vectors):
            branch = mt.grouped_matrix_product(mt.grouped_gated_product(normed, inner, offsets), outer, offsets)
            stream, normed = mt.gated_residual_norm(stream, branch, None, scale, weight_branch, weight_output)
        return normed

    def losses(self, species, offsets, targets):
        """Of each atom with a target (the others have -1)."""
        return mt.linear_cross_entropy(self(species, offsets), self.table, targets)


def atoms(n, species, environments, seed):
    """Atoms sorted by environment, whose species is the environment's favourite most of the time; a third of them are masked (species 0)."""
    gen = torch.Generator().manual_seed(seed)
    environment = torch.randint(environments, (n,), generator=gen).sort().values
    favourite = 1 + (environment * 7) % (species - 1)
    real = torch.where(torch.rand(n, generator=gen) < 0.8, favourite, torch.randint(1, species, (n,), generator=gen))
    masked = torch.rand(n, generator=gen) < 1 / 3
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(environment, minlength=environments).cumsum(0)])
    shown, targets = torch.where(masked, 0, real), torch.where(masked, real, -1)
    return [t.to(torch.int32).cuda() for t in (shown, offsets, targets)]


def step(model, data, optimizer, max_norm=1.0):
    """One training step; returns the mean loss and the norm of all gradients, on the device."""
    shown, offsets, targets = data
    loss, log_sum = model.losses(shown, offsets, targets)
    count = (targets >= 0).sum().clamp(min=1)
    mean = loss.sum() / count
    (mean + 1e-4 * log_sum.square().sum() / count).backward()
    norm = mt.clip_gradient_norm_([p.grad for p in model.parameters()], max_norm)
    optimizer.step()
    optimizer.zero_grad(set_to_none=True)
    return mean.detach(), norm


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--atoms", type=int, default=4096)
    ap.add_argument("--species", type=int, default=95)
    ap.add_argument("--environments", type=int, default=6)
    ap.add_argument("--channels", type=int, default=128)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--dtype", choices=DTYPE, default="bf16")
    a = ap.parse_args()
    model = MaskedSpecies(a.species, a.environments, a.channels, a.width, a.layers, DTYPE[a.dtype])
    optimizer = torch.optim.Adam(model.parameters(), 3e-3)
    for i in range(a.steps):
        loss, norm = step(model, atoms(a.atoms, a.species, a.environments, i), optimizer)
        if i % 50 == 0 or i == a.steps - 1:
            print(f"step {i}: loss {float(loss):.3f}, norm of the gradients {float(norm):.3f}")
    shown, offsets, targets = atoms(a.atoms, a.species, a.environments, a.steps)
    with torch.no_grad():
        loss, _ = model.losses(shown, offsets, targets)
        print(f"new atoms: {float((loss.sum() / (targets >= 0).sum()).exp()):.2f} species to choose from, on average")


if __name__ == "__main__":
    main()
