"""The example that runs the operators of the block together."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import species_blocks  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_learns(dtype):
    _, losses = species_blocks.train(steps=60, structures=16, atoms=50, dtype=dtype, species=7, channels=64, hidden=96)
    assert sum(losses[-10:]) < 0.5 * sum(losses[:10])


@pytest.mark.gpu
def test_one_atom_at_a_time_gives_what_all_together_give():
    """In f64: single rows go through other kernels than many."""
    model, _ = species_blocks.train(steps=2, structures=4, atoms=50, dtype=torch.float64, species=5, channels=48, hidden=80)
    generator = torch.Generator(device="cuda").manual_seed(1)
    species, charges, _, _ = species_blocks.batch(model, 3, 41, generator)
    with torch.no_grad():
        together = model(species, charges)
        alone = torch.cat([model(species[i:i + 1], charges[i:i + 1]) for i in range(0, 123, 5)])
    # (f64 up to the readout, which is in f32: sums of 48 terms)
    assert torch.allclose(alone, together[::5], rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_gradients_match_plain_torch():
    """The whole model's gradients, in f64, against the same model of plain operations."""
    torch.manual_seed(2)
    model = species_blocks.Model(species=6, channels=40, hidden=56, layers=2).to(device="cuda", dtype=torch.float64)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.1 * torch.randn_like(p))
    generator = torch.Generator(device="cuda").manual_seed(3)
    species, charges, _, _ = species_blocks.batch(model, 2, 90, generator)

    def plain():
        s = species.long()
        stream = model.table[s] * model.table.shape[1] ** 0.5 * (1 + charges[:, None].double())
        normed = stream
        for layer in model.layers:
            hidden = torch.nn.functional.silu(torch.einsum("rk,rkn->rn", normed, layer.widen[s]))
            branch = torch.einsum("rk,rkn->rn", hidden, layer.narrow[s])
            gate = torch.einsum("rk,rkn->rn", normed, layer.gate[s])
            unit = branch / torch.sqrt(branch.square().mean(1, keepdim=True) + 1e-5)
            stream = stream + layer.scale * torch.sigmoid(gate) * layer.weight_branch * unit
            normed = layer.weight_output * stream / torch.sqrt(stream.square().mean(1, keepdim=True) + 1e-5)
        return normed.float() @ model.readout.float()

    parameters = list(model.parameters())
    want = torch.autograd.grad(plain().sum(), parameters)
    got = torch.autograd.grad(model(species, charges).sum(), parameters)
    for g, w in zip(got, want):
        # the readout's rounding to f32 enters both in the same way; what is left is the order of sums in 64 bits, but for its own gradient
        assert (g - w).abs().max() <= 1e-5 * w.abs().max().clamp(min=1.0)
