"""The example of a model that guesses masked species: it runs, and its gradients are those of the same model written in plain
operations in 64 bits."""
import importlib.util
import math
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("masked_species", os.path.join(ROOT, "examples", "masked_species.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_loss(model, shown, offsets, targets):
    stream = model.table[shown.long()] * math.sqrt(model.table.shape[1])
    normed, bounds = stream, offsets.tolist()
    for inner, outer, (scale, weight_branch, weight_output) in zip(model.inner, model.outer, model.vectors):
        rows = []
        for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            u, v = (normed[lo:hi] @ inner[g]).chunk(2, 1)
            rows.append((u * torch.sigmoid(u) * v) @ outer[g])
        branch = torch.cat(rows)
        stream = stream + scale * weight_branch * branch / (branch.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
        normed = weight_output * stream / (stream.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
    keep = targets >= 0
    x = normed[keep] @ model.table.T
    log_sum = torch.logsumexp(x, 1)
    loss = log_sum - x.gather(1, targets[keep].long()[:, None])[:, 0]
    return loss.mean() + 1e-4 * log_sum.square().mean()


@pytest.mark.gpu
def test_gradients_are_those_of_plain_operations():
    """In float64, where the operators and the plain model differ by roundings alone: some 10^3 of them in a row, each of 2^-53, stay under 10^-11 of the
    largest value of a gradient."""
    module = example()
    torch.manual_seed(0)
    model = module.MaskedSpecies(20, 4, 24, 40, 2, torch.float64)
    shown, offsets, targets = module.atoms(300, 20, 4, 1)
    loss, log_sum = model.losses(shown, offsets, targets)
    count = (targets >= 0).sum()
    mine = torch.autograd.grad(loss.sum() / count + 1e-4 * log_sum.square().sum() / count, list(model.parameters()))
    plain = torch.autograd.grad(plain_loss(model, shown, offsets, targets), list(model.parameters()))
    for a, b in zip(mine, plain):
        assert (a - b).abs().max() <= 1e-11 * b.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_it_runs(dtype):
    module = example()
    model = module.MaskedSpecies(95, 5, 64, 96, 2, module.DTYPE[dtype])
    optimizer = torch.optim.Adam(model.parameters(), 1e-3)
    for i in range(3):
        loss, norm = module.step(model, module.atoms(700, 95, 5, i), optimizer, 0.5)
        assert loss.isfinite() and norm.isfinite() and norm > 0
    assert all(p.isfinite().all() for p in model.parameters())
