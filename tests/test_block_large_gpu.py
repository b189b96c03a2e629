"""The operators of the block on arrays of more than 2^31 values: what lies behind that is where it should be."""
import pytest
import torch

import mops_b200.torch as mt

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [300, 20000])
def test_a_large_table(tokens):
    V, D = 1_100_003, 2048
    assert V * D > 2 ** 31
    W = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    indices = (torch.arange(tokens, device="cuda") * 7919 % V).to(torch.int32)
    indices[-2:] = V - 1
    W[indices.long()] = (indices % 97).to(torch.bfloat16)[:, None]
    W.requires_grad_(True)
    output = mt.embedding_lookup(W, indices, 2.0)
    assert torch.equal(output.detach(), W.detach()[indices.long()] * 2)
    got, = torch.autograd.grad(output, [W], torch.ones_like(output))
    rows, counts = torch.unique(indices, return_counts=True)
    assert torch.equal(got[rows.long()], (2 * counts)[:, None].expand(-1, D).to(torch.bfloat16))
    got[rows.long()] = 0
    assert not got.any()


@pytest.mark.parametrize("dtype,K,N", [(torch.bfloat16, 2112, 24), (torch.bfloat16, 24, 2112), (torch.bfloat16, 2111, 19), (torch.float32, 2112, 24), (torch.float32, 24, 2112)])
def test_many_rows_of_a_product(dtype, K, N):
    """The second half of the rows is the first half with its values doubled: its results are the first half's, doubled, bit for bit."""
    half = 524_288
    R = 2 * half
    assert R * max(K, N) > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(1)
    A, grad = torch.empty(R, K, dtype=dtype, device="cuda"), torch.empty(R, N, dtype=dtype, device="cuda")
    for t in (A, grad):
        t[:half] = torch.randn(half, t.shape[1], generator=gen, device="cuda", dtype=dtype)
        torch.mul(t[:half], 2, out=t[half:])
    W = torch.randn(2, K, N, generator=gen, device="cuda", dtype=dtype)
    W[1] = W[0]
    offsets = torch.tensor([0, half, R], dtype=torch.int32, device="cuda")
    A.requires_grad_(True), W.requires_grad_(True)
    output = mt.grouped_matrix_product(A, W, offsets)
    gA, gW = torch.autograd.grad(output, [A, W], grad)
    for t in (output.detach(), gA):
        assert torch.equal(t[half:], t[:half] * 2) and t[-1].any()
    assert torch.equal(gW[1], gW[0] * 4) and gW[0].any()
    few = slice(R - 3, R)
    want = A.detach()[few].double() @ W.detach()[1].double()
    assert ((output.detach()[few].double() - want).abs().max() / want.abs().max()) < 0.01


def test_large_matrices():
    """Matrices of more than 2^31 values together, a few rows and many."""
    G, K, N = 1030, 1024, 2048
    assert G * K * N > 2 ** 31
    W = torch.empty(G, K, N, dtype=torch.bfloat16, device="cuda")
    W.copy_((torch.arange(G, device="cuda") % 64).to(torch.bfloat16)[:, None, None].expand(G, K, N))
    for rows in (12, 700):
        A = torch.ones(rows, K, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
        offsets = torch.zeros(G + 1, dtype=torch.int32, device="cuda")
        offsets[G - 1], offsets[G] = rows // 3, rows  # two thirds of the rows have the last matrix, the others the one before
        leaf = W.detach().requires_grad_(True)
        output = mt.grouped_matrix_product(A, leaf, offsets)
        value = torch.where(torch.arange(rows, device="cuda") < rows // 3, (G - 2) % 64, (G - 1) % 64)
        assert torch.equal(output.detach(), (value * K).to(torch.bfloat16)[:, None].expand(rows, N))
        gA, gW = torch.autograd.grad(output, [A, leaf], torch.ones_like(output))
        assert torch.equal(gA, (value * N).to(torch.bfloat16)[:, None].expand(rows, K))
        assert (gW[G - 1] == rows - rows // 3).all() and (gW[G - 2] == rows // 3).all() and not gW[:G - 2].any()


@pytest.mark.parametrize("C", [8192, 8193])
def test_many_rows_of_a_norm(C):
    """The second half of the rows is the first half again."""
    half = 131_200
    R = 2 * half
    assert R * C > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(2)

    def rows():
        t = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
        t[:half] = torch.randn(half, C, generator=gen, device="cuda", dtype=torch.bfloat16)
        t[half:] = t[:half]
        return t

    x, b = rows().requires_grad_(True), rows().requires_grad_(True)
    s, w, p = (torch.ones(C, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    outputs = mt.gated_residual_norm(x, b, None, s, w, p, 1e-5)
    grads = [rows(), rows()]
    for t in [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, [x, b], grads)):
        assert torch.equal(t[half:], t[:half]) and t[-1].any()
    want = x.detach()[-1].double() + b.detach()[-1].double() / (b.detach()[-1].double().square().mean() + 1e-5).sqrt()
    assert ((outputs[0].detach()[-1].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
