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


# ------------------------------------------------------------------------------------ many rows
def exactly(arguments, epsilon, grads):
    """Both outputs and all gradients in 64 bits, and for each value the sum T of the magnitudes of the terms that it is made of: every difference is
    replaced by a sum, and where a root's relative error is that of a sum of squares of such values, by as much more (kappa)."""
    x, b, g, s, w, p = (None if t is None else t.detach().double() for t in arguments)
    gs, gh = (t.double() for t in grads)
    mean = lambda t: t.mean(1, keepdim=True)
    z, o = (torch.ones_like(x[:, :1]), torch.zeros_like(x[:, :1])) if g is None else (torch.sigmoid(g), torch.sigmoid(-g))
    q = (mean(b * b) + epsilon).rsqrt()
    n = b * q
    branch = s * w * z * n
    y, Y = x + branch, x.abs() + branch.abs()
    r = (mean(y * y) + epsilon).rsqrt()
    kappa = 1 + mean(Y * Y) * r * r
    ph = p * gh
    ds = gs + r * ph - y * r ** 3 * mean(ph * y)
    D = gs.abs() + kappa * (r * ph.abs() + 3 * Y * r ** 3 * mean(ph.abs() * Y))
    dn, N = ds * s * w * z, D * (s * w).abs() * z
    values = [y, p * y * r, ds, q * (dn - n * mean(dn * n))]
    terms = [Y, p.abs() * Y * r * kappa, D, q * (N + n.abs() * mean(N * n.abs()))]
    if g is not None:
        full, F = dn * n * o, N * n.abs() * o
        values.append(full if g.shape[1] == x.shape[1] else full.sum(1, keepdim=True))
        terms.append(F if g.shape[1] == x.shape[1] else F.sum(1, keepdim=True))
    P, Q = (ds * z * n).sum(0), (D * z * n.abs()).sum(0)
    values += [w * P, s * P, (gh * y * r).sum(0)]
    terms += [w.abs() * Q, s.abs() * Q, (gh.abs() * Y * r * kappa).sum(0)]
    return values, terms


def bounds(values, terms, arguments):
    """A sum over a row is a chain of at most C / 256 + 16 additions in a thread and as many as a tree of threads and warps has, 24; a sum over rows one of the rows of a team
    (there are 148 of them at least, where there are so many rows), of the blocks, over 128 parts, and a tree. Such sums enter a value one within the other, four of them at most, each
    with a few products besides; twice that is allowed, and the gates of 16-bit types have 8 + 4 |gate| units more (approximate exponentials)."""
    R, C = arguments[0].shape
    dtype = arguments[0].dtype
    row = C / 256 + 40 + 16
    if arguments[2] is not None and dtype in (torch.float16, torch.bfloat16):
        row += 8 + 4 * float(arguments[2].detach().abs().max())
    rows = row + R / 148 + 1 + 148 * 16 / 128 + 16
    return [ROUND[dtype] * v.abs() + 8 * (rows if v.dim() == 1 else row) * SUM[dtype] * t + SMALLEST[dtype] for v, t in zip(values, terms)]


NAMES = ["stream", "normed", "grad_residual", "grad_branch", "grad_gate", "grad_scale", "grad_weight_branch", "grad_weight_output"]
MANY_ROWS = [(30011, 40), (9001, 250), (6007, 1024), (4003, 1002), (1501, 4096), (1301, 4099), (1903, 8200)]


def problem(R, C, gate, dtype, device):
    gen = torch.Generator(device=device).manual_seed(R + C)
    draw = lambda shape, size: (torch.randn(shape, generator=gen, device=device, dtype=torch.float64) * size).to(dtype)
    arguments = [draw((R, C), 2.0), draw((R, C), 1.0), None if gate == 0 else draw((R, 1 if gate == 1 else C), 2.0)]
    arguments += [(draw((C,), 0.2) + 1).to(dtype) for _ in range(3)]
    return arguments, [draw((R, C), 1.0), draw((R, C), 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [0, 1, 2])
@pytest.mark.parametrize("R,C", MANY_ROWS)
def test_blocks_walk_over_many_rows(dtype, gate, R, C):
    """At least three rows for every block, or warp, that fits the GPU: places of rings and rows fetched ahead are used again, sums stay over rows."""
    arguments, grads = problem(R, C, gate, dtype, "cuda")
    leaves = [t.requires_grad_(True) for t in arguments if t is not None]
    outputs = mt.gated_residual_norm(*arguments, 1e-5)
    got = [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, leaves, grads))
    values, terms = exactly(arguments, 1e-5, grads)
    names = [n for n in NAMES if gate or n != "grad_gate"]
    for g, v, b, name in zip(got, values, bounds(values, terms, arguments), names):
        error = (g.double() - v).abs()
        assert g.shape == v.shape and not (error > b).any() and not error.isnan().any(), f"{name}: {(error / b).max().item():.2f} of the bound"


@pytest.mark.parametrize("gate", [0, 1, 2])
@pytest.mark.parametrize("R,C", [(700, 40), (400, 250), (300, 1002), (60, 4099), (40, 8200)])
def test_bounds_are_too_small_for_a_row_left_out(gate, R, C):
    """On the host: results of zeros, and sums over rows without one of the rows, are outside of the bounds, in every type. And the formulas' gradients are those of the
    outputs."""
    for dtype in DTYPES:
        arguments, grads = problem(R, C, gate, dtype, "cpu")
        values, terms = exactly(arguments, 1e-5, grads)
        limits = bounds(values, terms, arguments)
        assert all((v.abs() > b).double().mean() > 0.5 for v, b in zip(values, limits))
        for row in (0, R // 2, R - 1):
            keep = torch.arange(R) != row
            less = [t if t is None or t.dim() == 1 else t[keep] for t in arguments]
            without, _ = exactly(less, 1e-5, [t[keep] for t in grads])
            for v, x, b in list(zip(values, without, limits))[-3:]:
                assert ((v - x).abs() > b).any()  # (one value is enough for a test to fail)
    leaves = [t.double().requires_grad_(True) for t in arguments if t is not None]
    it = iter(leaves)
    x, b, g, s, w, p = (None if t is None else next(it) for t in arguments)
    y = x + s * w * (1.0 if g is None else torch.sigmoid(g)) * b / (b.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
    h = p * y / (y.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
    for d, v, t in zip(torch.autograd.grad([y, h], leaves, [t.double() for t in grads]), values[2:], terms[2:]):
        assert ((d - v).abs() <= 1e-12 * t).all()
