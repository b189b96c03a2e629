"""Scratch memory of calls that end with an exception."""
import pytest
import torch

from mops_b200 import _lib


def array(t):
    return _lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), t.stride())


@pytest.mark.gpu
def test_a_refused_call_gives_its_scratch_memory_back():
    """2^30 groups of one value each are refused, as there would be more tiles than a grid has blocks, when the operands have been copied
    already (64 MB each, as their rows begin anywhere). The refusals that follow find that memory free again."""
    groups, rows = 1 << 30, 1 << 22
    grad_W = torch.empty(groups, 1, 1, dtype=torch.bfloat16, device="cuda")
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    A, grad = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    left = []
    for _ in range(8):
        with pytest.raises(_lib.MopsError, match="the number of tiles"):
            _lib.call("mops_b200_cuda_grouped_matrix_product_vjp", [_lib.Array(), array(grad_W), array(grad), array(A), array(grad_W), array(offsets)])
        torch.cuda.synchronize()
        left.append(torch.cuda.mem_get_info()[0])
    del grad_W, offsets
    torch.cuda.empty_cache()
    assert left[1] - left[-1] < 64 << 20
