"""gated_residual_norm where it can go wrong and small mistakes show: gates far from zero, blocks that walk over many rows, sums over rows
and columns. Against the formulas in 64 bits, with bounds value by value."""
import pytest
import torch

import mops_b200.torch as mt
from test_block_ops import DTYPES, ROUND, SMALLEST, SUM, normal


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("C", [40, 129, 1024, 1002, 2056, 20000])
def test_gate_gradients_of_large_gates(dtype, per_row, C):
    """The gradient of a gate is proportional to z (1 - z), z = sigmoid(gate), which is e^-|gate| for large gates of either sign.

    All of its factors are positive here, and it has no terms of the second output (whose gradient is zero), so it is a product: of the
    root of a sum of C squares, of three given factors and of z and 1 - z, and for a gate per row a sum of C such. Its relative error is that of the sums, (C + 1) u
    each, of some twenty more roundings, and of the exponential: 2 units for the library's, 2^-21 + |gate| 2^-22 for the approximate instructions of 16-bit types.
    """
    R = 24
    gate = torch.cat([torch.tensor([8.0, 10.0, 12.0, 14.0, 15.0, 16.0, 17.0, 18.0, 20.0, 25.0], dtype=torch.float64), -torch.arange(1.0, 25.0, 3, dtype=torch.float64),
                      torch.zeros(6, dtype=torch.float64)])[:R, None].cuda()
    if not per_row:
        gate = gate + 0.25 * torch.rand(R, C, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(1))
    gate = gate.to(dtype)
    branch, residual = normal((R, C), dtype, 2), normal((R, C), dtype, 3)
    size = 0.5 + torch.rand(R, C, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(4))
    grad = (branch.double().sign() * size * 64).to(dtype)
    scale, weight_branch, weight_output = ((normal((C,), dtype, 5 + i) * 0.1 + 1).clamp(0.5, 1.5) for i in range(3))
    gate.requires_grad_(True)
    stream, normed = mt.gated_residual_norm(residual, branch, gate, scale, weight_branch, weight_output, 1e-5)
    got, = torch.autograd.grad([stream, normed], [gate], [grad, torch.zeros_like(grad)])
    b, g = branch.double(), gate.detach().double()
    want = grad.double() * scale.double() * weight_branch.double() * b / (b.square().mean(1, keepdim=True) + 1e-5).sqrt()
    want = want * torch.sigmoid(g) * torch.sigmoid(-g)
    if per_row:
        want = want.sum(1, keepdim=True)
    u = SUM[dtype]
    relative = ROUND[dtype] + (2 * (C + 1) + 20) * u
    if dtype in (torch.float16, torch.bfloat16):
        relative = relative + 2.0 ** -21 + g.abs() * 2.0 ** -22
    error = (got.double() - want).abs()
    inside = want.to(dtype).isfinite()  # (in f16 sums over long rows go beyond the type)
    assert (want >= 0).all() and torch.equal(got.isfinite(), inside) and inside.any()
    assert not (error > relative * want + SMALLEST[dtype])[inside].any(), (error / want)[inside].nan_to_num(0).max().item()
