"""grouped_gated_product on shapes of which one dimension has a size of 1, stored either way round."""
import pytest
import torch

from test_training_ops import check_gated, normal, offsets_of


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,N", [([33], 1), ([1], 1), ([485], 1), ([40, 0, 3, 100], 2), ([63], 5), ([3] * 20, 12), ([300], 8), ([700], 3), ([200, 1], 130)])
@pytest.mark.parametrize("gap", [0, 1, 7])
def test_matrices_of_one_row_whose_columns_lie_apart(dtype, rows, N, gap):
    W = normal((len(rows), 2 * N, 1 + gap), dtype, 1, 2.0)[:, :, gap:].transpose(1, 2)
    assert W.shape == (len(rows), 1, 2 * N)
    check_gated(normal((sum(rows), 1), dtype, 2), W, offsets_of(rows), normal((sum(rows), N), dtype, 3), "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,K", [([1], 1), ([33], 7), ([400, 3], 130), ([1200], 16)])
@pytest.mark.parametrize("gap", [0, 1])
def test_layers_of_one_column(dtype, rows, K, gap):
    R = sum(rows)
    for W in (normal((len(rows), 2, K + gap), dtype, 1, K ** -0.5)[:, :, gap:].transpose(1, 2), normal((len(rows), K, 2 + gap), dtype, 1, K ** -0.5)[:, :, gap:]):
        check_gated(normal((R, K + gap), dtype, 2)[:, gap:], W, offsets_of(rows), normal((R, 1 + gap), dtype, 3)[:, gap:])
