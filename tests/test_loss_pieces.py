"""linear_cross_entropy where its gradients are taken in several pieces of the vocabulary: the last one may be of any size, and the
depth of its products is cut as that of the others is. Against a plain implementation in 64 bits, some rows at a time; tolerances as in
test_training_ops.py, with the sums over all rows counted as such.
"""
import ctypes

import pytest
import torch

import mops_b200
import mops_b200.torch as mt
from mops_b200 import _lib

from test_training_ops import inner_round, normal, some_targets, unit, within

MOST = 40_000_000  # logits of the rows that the plain implementation takes at a time


def plain_in_blocks(A, W, targets, scale, grad_loss, grad_log_sum):
    """Values and bounds of (loss, log_sum, grad_A, grad_W); rows whose target is -1 have none."""
    u, v = unit(A.dtype), inner_round(A.dtype)
    small = {torch.float16: 2.0 ** -36, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[A.dtype]
    small *= 1 + float((grad_loss.abs() + grad_log_sum.abs()).max())
    R, (V, C) = A.shape[0], W.shape
    W = W.double()
    W_size = W.abs()
    sums = A.new_zeros(R, dtype=torch.float64)
    rows = A.new_zeros((R, C), dtype=torch.float64)
    loss, log_sum, grad_A, e_loss_all, e_sum_all, e_A = sums, sums.clone(), rows, sums.clone(), sums.clone(), rows.clone()
    grad_W, e_W = torch.zeros_like(W), torch.zeros_like(W)
    for r in torch.arange(R, device=A.device).split(max(1, MOST // V)):
        keep = targets[r] != -1
        t = torch.where(keep, targets[r], 0).long()[:, None]
        a = torch.where(keep[:, None], A[r].double(), 0.0)
        x = scale * (a @ W.T)
        ex = scale * 4 * (C + 4) * u * (a.abs() @ W_size.T) + 4 * u * x.abs()
        top = torch.logsumexp(x, 1)
        x_t = x.gather(1, t)[:, 0]
        e_sum = ex.amax(1) + (400 + V / 64) * u + 4 * u * top.abs()
        e_loss = e_sum + ex.gather(1, t)[:, 0] + 4 * u * (top.abs() + x_t.abs())
        gl, gs = (torch.where(keep, g[r].double(), 0.0)[:, None] for g in (grad_loss, grad_log_sum))
        dx = (gl + gs) * torch.exp(x - top[:, None])
        e_dx = dx.abs() * (ex + e_sum[:, None] + 32 * u * (1 + (x - top[:, None]).abs()))
        e_dx.scatter_add_(1, t, dx.gather(1, t).abs() * 2 * e_loss[:, None] + 4 * u * gl.abs())
        dx.scatter_add_(1, t, -gl)
        e_dx += v * (dx.abs() + e_dx) + small
        e_dx *= keep[:, None]
        dx_size = dx.abs()
        loss[r], log_sum[r] = torch.where(keep, top - x_t, 0.0), torch.where(keep, top, 0.0)
        e_loss_all[r], e_sum_all[r] = keep * e_loss, keep * e_sum
        grad_A[r] = scale * dx @ W
        e_A[r] = scale * (e_dx @ W_size + 4 * (V + 4) * u * (dx_size @ W_size))
        grad_W += scale * dx.T @ a
        e_W += scale * (e_dx.T @ a.abs() + 4 * (R + 4) * u * (dx_size.T @ a.abs()))
    return (loss, log_sum, grad_A, grad_W), (e_loss_all, e_sum_all, e_A, e_W)


def leave_nan(dtype):
    """A call whose sums are NaN: they stay in tensor memory and in workspaces."""
    leaves = [torch.full((3000, 264), float("nan"), dtype=dtype, device="cuda").requires_grad_(True), normal((6000, 264), dtype, 2, 0.125).requires_grad_(True)]
    loss = mt.linear_cross_entropy(*leaves, some_targets(3000, 6000, 1.0))[0]
    assert torch.autograd.grad(loss.sum(), leaves)[0].isnan().all()


def check_pieces(dtype, R, V, C, kept=0.9, scale=1.25):
    A, W = normal((R, C), dtype, 1, 2.0).requires_grad_(True), normal((V, C), dtype, 2, C ** -0.5).requires_grad_(True)
    targets = some_targets(R, V, kept)
    targets[R // 2] = V - 1  # (in the last piece)
    grads = [normal((R,), torch.float32, 9 + i) for i in range(2)]
    leave_nan(dtype)
    outputs = mt.linear_cross_entropy(A, W, targets, scale)
    got = [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, [A, W], grads))
    values, errors = plain_in_blocks(A.detach(), W.detach(), targets, scale, *grads)
    for g, w, e, what in zip(got, values, errors, ("loss", "log_sum", "grad_A", "grad_W")):
        within(g, w, e, what)
    again = mt.linear_cross_entropy(A, W, targets, scale)
    for a, b in zip(list(again) + list(torch.autograd.grad(again, [A, W], grads)), got):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,V,C", [(3552, 56840, 8), (2048, 113672, 64), (12288, 19144, 64), (4196, 118267, 48), (14662, 18650, 24), (10298, 19006, 35),
                                   (8079, 18965, 640), (3552, 56833, 33), (6000, 151669, 1024)])
def test_gradients_whose_last_piece_has_fewer_stages_than_slices(dtype, R, V, C):
    check_pieces(dtype, R, V, C)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,C", [
    (torch.bfloat16, 8192, 40000, 16), (torch.float16, 3000, 113700, 40), (torch.bfloat16, 20000, 18945, 72),
    (torch.float32, 2100, 40000, 128), (torch.float32, 2100, 28673, 130)])
def test_gradients_of_several_pieces(dtype, R, V, C):
    check_pieces(dtype, R, V, C)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,V,pieces", [(1, 2200000, 3), (128, 1100003, 2), (129, 1100003, 3), (256, 1100003, 3), (300, 1100003, 3)])
def test_gradients_of_few_rows_of_a_very_large_table(dtype, R, V, pieces):
    """dx has room up to the end of a tile, for two parts of up to 256 rows each: half a GB at the most, however few the rows are."""
    A, W, targets = normal((R, 8), dtype, 1, 2.0), normal((V, 8), dtype, 2, 0.35), some_targets(R, V, 1.0)
    targets[R // 2] = V - 1
    loss, log_sum = mops_b200.linear_cross_entropy(A, W, targets)
    grads = [normal((R,), torch.float32, 9 + i) for i in range(2)]
    got_A, got_W = torch.empty_like(A), torch.empty_like(W)
    arrays = [_lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), t.stride())
              for t in (got_A, got_W, *grads, loss, log_sum, A, W, targets)]
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    _lib.call("mops_b200_cuda_linear_cross_entropy_vjp", arrays + [ctypes.c_double(1.0), ctypes.c_int64(-1)])
    torch.cuda.synchronize()
    assert any(f", {pieces} pieces" in k for k in _lib.last_kernels()), _lib.last_kernels()
    assert before - torch.cuda.mem_get_info()[0] < 640 << 20
    values, errors = plain_in_blocks(A, W, targets, 1.0, *grads)
    for g, w, e, what in zip((loss, log_sum, got_A, got_W), values, errors, ("loss", "log_sum", "grad_A", "grad_W")):
        within(g, w, e, what)
