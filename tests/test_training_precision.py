"""Gradients of few rows in 16 bits, where the errors of what is rounded on its way into products do not average out: the loss keeps the gradients
of logits of up to 256 rows in two parts of 16 bits, the gated layer computes up to 2048 values of dU and dV in 32 bits. The bounds of
test_training_ops.py, with what these paths round in the place of one rounding to 16 bits: what is left of a value in two parts is off by v of the rest, which is at most v of the value, so
by v^2 of it; dU and dV are not rounded (the products of f32 in three parts are within the factor of 4 of their sums).

Bounds value by value allow for the worst sums. What errors come to on average tells a path that rounds once from one that rounds twice, whose errors are some 1.4 times as large: a result that is off by e before it is
rounded is off by no more than its rounding and 2 e. Terms that are off by 4 u each, with signs of their own, make sums of n that are off by some 4 sqrt(n) u of their root mean square: of 1000 to 4000 terms by
2^-17, where the rounding is 0.3 * 2^-11 on average, or more; together, as squares, less than 1.02 times the rounding. The bound is 1.1.
"""
import pytest
import torch

import mops_b200.torch as mt
import test_training_ops
from test_training_ops import ROUND, check_gated, check_loss, gated_plain, loss_plain, normal, offsets_of, some_targets

DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C,kept", [(1, 3001, 264, 1.0), (5, 40, 8, 1.0), (17, 5003, 130, 0.8), (128, 1000, 72, 0.9), (129, 3001, 264, 0.9), (256, 9001, 520, 1.0)])
def test_loss_of_up_to_256_rows(monkeypatch, dtype, R, V, C, kept):
    monkeypatch.setattr(test_training_ops, "inner_round", lambda dtype: ROUND[dtype] ** 2)
    check_loss(normal((R, C), dtype, 1, 2.0), normal((V, C), dtype, 2, C ** -0.5), some_targets(R, V, kept), 1.25)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,K,N", [([1], 2048, 1024), ([3, 0, 1], 264, 256), ([9, 7], 33, 64), ([1, 1, 30], 1000, 32), ([1024], 40, 1)])
def test_gated_of_up_to_2048_values(monkeypatch, dtype, activation, rows, K, N):
    monkeypatch.setattr(test_training_ops, "inner_round", lambda dtype: 0.0)
    R = sum(rows)
    assert R * 2 * N <= 2048
    check_gated(normal((R, K), dtype, 1), normal((len(rows), K, 2 * N), dtype, 2, 2 * K ** -0.5), offsets_of(rows), normal((R, N), dtype, 3), activation)


def rounded_once(got, want):
    """The errors' root mean square over that of results that are rounded once."""
    return float((got.double() - want).square().mean().sqrt() / (want.to(got.dtype).double() - want).square().mean().sqrt())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C", [(128, 1000, 264), (130, 3001, 72), (256, 3001, 264)])
def test_loss_of_up_to_256_rows_is_rounded_once(dtype, R, V, C):
    A, W, targets = normal((R, C), dtype, 1, 2.0).requires_grad_(True), normal((V, C), dtype, 2, C ** -0.5).requires_grad_(True), some_targets(R, V, 1.0)
    grads = [normal((R,), torch.float32, 9 + i) for i in range(2)]
    got = torch.autograd.grad(mt.linear_cross_entropy(A, W, targets, 1.25), [A, W], grads)
    want = loss_plain(A.detach(), W.detach(), targets, 1.25, -1, *grads)[0][2:]
    for g, w in zip(got, want):
        assert rounded_once(g, w) < 1.1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,K,N", [([1], 2048, 1024), ([3, 0, 1], 264, 256), ([9, 7], 330, 64), ([1, 1, 30], 1000, 32)])
def test_gated_of_up_to_2048_values_is_rounded_once(dtype, activation, rows, K, N):
    A, W = normal((sum(rows), K), dtype, 1).requires_grad_(True), normal((len(rows), K, 2 * N), dtype, 2, 2 * K ** -0.5).requires_grad_(True)
    offsets, grad = offsets_of(rows), normal((sum(rows), N), dtype, 3)
    got = torch.autograd.grad(mt.grouped_gated_product(A, W, offsets, activation), [A, W], grad)
    want = gated_plain(A.detach(), W.detach(), offsets, grad, activation)[0][1:]
    for g, w in zip(got, want):
        assert rounded_once(g, w) < 1.1
