"""Grouped products of matrices that have to be copied, as their rows begin anywhere, and have few rows, or few columns, that are long."""
import pytest
import torch

import mops_b200.torch as mt

pytestmark = pytest.mark.gpu


def whole_numbers(shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("G,K,N", [(1, 3, 30011), (1, 16, 20003), (2, 5, 8185), (1, 1, 4099), (3, 33, 1021), (1, 2, 513), (1, 7, 50009)])
@pytest.mark.parametrize("other_way", [False, True])
def test_rows_picked_out_of_matrices(dtype, G, K, N, other_way):
    """Each row of A picks a row of its group's matrix, or a multiple of it."""
    W = whole_numbers((G, N, K + 1), dtype, 1)[:, :, 1:].transpose(1, 2) if other_way else whole_numbers((G, K, N + 2), dtype, 1)[:, :, 1:N + 1]
    R = 300
    offsets = torch.linspace(0, R, G + 1).to(torch.int32).cuda()
    row = torch.arange(R, device="cuda")
    group = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=G - 1)
    A = torch.zeros(R, K, dtype=dtype, device="cuda")
    A[row, row % K] = (1.0 + row % 3).to(dtype)
    got = mt.grouped_matrix_product(A, W, offsets)
    assert torch.equal(got, W[group, row % K] * (1.0 + row % 3)[:, None].to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_long_rows(dtype):
    R, K, N = 130, 5, 20011
    A, W, grad = whole_numbers((R, K), dtype, 1), whole_numbers((1, K, N), dtype, 2), torch.zeros(R, N, dtype=dtype, device="cuda")
    column = torch.arange(R, device="cuda") * 151
    grad[torch.arange(R, device="cuda"), column] = 1.0
    A.requires_grad_(True), W.requires_grad_(True)
    output = mt.grouped_matrix_product(A, W, torch.tensor([0, R], dtype=torch.int32, device="cuda"))
    grad_A, grad_W = torch.autograd.grad(output, [A, W], grad)
    assert torch.equal(grad_A, W.detach()[0, :, column].T)
    want = torch.zeros_like(W)
    want[0, :, column] = A.detach().T
    assert torch.equal(grad_W, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_copies_of_few_long_rows_use_all_of_the_device(dtype):
    """They take little of the whole call; by a few blocks alone the call took six times as long as one without copies."""
    def shortest(N):
        A, W, offsets = whole_numbers((300, 3), dtype, 1), whole_numbers((1, 3, N), dtype, 2), torch.tensor([0, 300], dtype=torch.int32, device="cuda")
        times = []
        for _ in range(12):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            mt.grouped_matrix_product(A, W, offsets)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)
    assert shortest(500001) < 3.5 * shortest(500032)  # (1.6 to 2, as rows of an odd width are also written value by value)
