"""What a training step has behind the operators of the block: grouped_gated_product, linear_cross_entropy and the norm of
gradients. Refusals on the CPU; on the GPU forward and gradients against a plain implementation in 64 bits, and gradients
against differences.

Tolerances, value by value, to first order, with u the unit roundoff of the sums' type (2^-24, f64: 2^-53) and v that of the
output's (f16 2^-11, bf16 2^-8):

* a sum of n products of exact operands is off by at most 4 (n + 4) u sum|terms| (the factor of 4 covers sums that are truncated where they
  would be rounded, and f32 products in three parts);
* a function of a value that is off by e is off by e times its steepest slope (silu, gelu: 1.2, and their slopes: 1.2 as well), and by
  32 (1 + |x|) u of its own;
* what is rounded to 16 bits on its way into a product (dU, dV, dx) is off by v of itself, and the product by the sum of these times |the other operand|.
"""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import mops_b200
import mops_b200.torch as mt

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
ROUND = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 1e-44, torch.float64: 1e-320, torch.float16: 6e-8, torch.bfloat16: 1e-40}


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def inner_round(dtype):
    """Of what goes into a second product."""
    return ROUND[dtype] if dtype in (torch.float16, torch.bfloat16) else 0.0


def within(got, want, error, what=""):
    """|got - want| <= v |want| + error, value by value."""
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    if not got.numel():
        return
    bound = ROUND[got.dtype] * want.abs() * (1 + 2.0 ** -6) + error + SMALLEST[got.dtype]
    off = (got.double() - want).abs()
    # a value that is half a step above the type's largest (2^16 - 16 in f16, whose largest is 2^16 - 32) rounds to infinity
    largest = torch.finfo(got.dtype).max * (1 + 0.5 * ROUND[got.dtype])
    off = torch.where(got.isinf() & (got.sign() == want.sign()) & (want.abs() + error >= largest), 0.0, off)
    assert not off.isnan().any() and not (off > bound).any(), f"{what}: over the bound by {(off - bound).max().item():.3e}"


def normal(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * scale).to(dtype)


def offsets_of(rows):
    return torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")


def library_array(t):
    from mops_b200 import _lib
    return _lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), t.stride())


# =============================================================================== refusals
def test_schemas():
    schemas = {
        "grouped_gated_product": 'mops::grouped_gated_product(Tensor A, Tensor W, Tensor offsets, str activation="silu") -> Tensor',
        "linear_cross_entropy": "mops::linear_cross_entropy(Tensor A, Tensor W, Tensor targets, float scale=1., int ignore_index=-1) "
                                "-> (Tensor loss, Tensor log_sum)",
        "gradient_norm": "mops::gradient_norm(Tensor[] gradients) -> Tensor",
        "clip_gradient_norm": "mops::clip_gradient_norm(Tensor[] gradients, float max_norm) -> (Tensor norm, Tensor[] clipped)",
        "clip_gradient_norm_": "mops::clip_gradient_norm_(Tensor(a!)[] gradients, float max_norm) -> Tensor",
    }
    for name, schema in schemas.items():
        assert str(getattr(torch.ops.mops, name).default._schema) == schema


def test_operators_refuse_wrong_arguments():
    A, W, o = torch.zeros(5, 4), torch.zeros(1, 4, 6), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="grouped_gated_product is not implemented for device cpu"):
        mt.grouped_gated_product(A, W, o)
    with pytest.raises(ValueError, match="activation must be one of silu, gelu in grouped_gated_product, found relu"):
        mt.grouped_gated_product(A, W, o, "relu")
    with pytest.raises(TypeError, match="All floating point tensors must be of the same dtype"):
        mt.grouped_gated_product(A, W.half(), o)
    with pytest.raises(TypeError, match="All index tensors must be of type int32"):
        mt.grouped_gated_product(A, W, o.long())
    with pytest.raises(ValueError, match="Expected W to have 3 dimensions"):
        mt.grouped_gated_product(A, A, o)
    T, t = torch.zeros(7, 4), torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="linear_cross_entropy is not implemented for device cpu"):
        mt.linear_cross_entropy(A, T, t)
    with pytest.raises(TypeError, match="All index tensors must be of type int32"):
        mt.linear_cross_entropy(A, T, t.long())
    with pytest.raises(TypeError, match="All floating point tensors must be of the same dtype"):
        mt.linear_cross_entropy(A, T.double(), t)
    with pytest.raises(ValueError, match="Expected targets to have 1 dimensions"):
        mt.linear_cross_entropy(A, T, t[:, None])
    for f in (mt.gradient_norm, lambda g: mt.clip_gradient_norm(g, 1.0), lambda g: mt.clip_gradient_norm_(g, 1.0)):
        with pytest.raises(ValueError, match="no gradients in"):
            f([])
        with pytest.raises(ValueError, match="is not implemented for device cpu"):
            f([A, W])
        with pytest.raises(TypeError, match="only float32, float64, float16 and bfloat16 are supported"):
            f([A, o])
        with pytest.raises(NotImplementedError, match="derivatives are not supported"):
            f([A.clone().requires_grad_(True)])


def test_front_end_refuses_wrong_arguments():
    A, W, o, t = np.zeros((5, 4)), np.zeros((1, 4, 6)), np.zeros(2, np.int32), np.zeros(5, np.int32)
    with pytest.raises(ValueError, match="`W` must be a 3D array in grouped_gated_product"):
        mops_b200.grouped_gated_product(A, A, o)
    with pytest.raises(ValueError, match="`activation` must be one of silu, gelu in grouped_gated_product_vjp, got 'tanh'"):
        mops_b200.grouped_gated_product_vjp(A, A, W, o, "tanh")
    with pytest.raises(TypeError, match="Wrong dtype for targets in linear_cross_entropy"):
        mops_b200.linear_cross_entropy(A, A, A[:, 0])
    with pytest.raises(TypeError, match="`scale` must be a number in linear_cross_entropy"):
        mops_b200.linear_cross_entropy(A, A, t, None)
    with pytest.raises(ValueError, match="`loss` must be a 1D array in linear_cross_entropy_vjp"):
        mops_b200.linear_cross_entropy_vjp(None, None, A, t, A, A, t)
    with pytest.raises(ValueError, match="no gradients in gradient_norm"):
        mops_b200.gradient_norm([])
    with pytest.raises(TypeError, match="`gradients` must be arrays in clip_gradient_norm"):
        mops_b200.clip_gradient_norm([1.0], 1.0)
    with pytest.raises(TypeError, match="`max_norm` must be a number in clip_gradient_norm"):
        mops_b200.clip_gradient_norm([A], "1")


def _array(shape, dtype="float32", stride=None, data=0x1000):
    """An array that is never read: shapes are checked before anything is launched."""
    from mops_b200 import _lib
    if stride is None:
        stride = [int(np.prod(shape[d + 1:])) for d in range(len(shape))]
    return _lib.make_array(data, dtype, shape, stride)


_o3, _t7 = _array((3,), "int32"), _array((7,), "int32")


def _loss(**changed):
    a = dict(loss=_array((7,)), log_sum=_array((7,)), A=_array((7, 4)), W=_array((9, 4)), targets=_t7, scale=1.0, ignore=-1)
    a.update(changed)
    return list(a.values())


def _loss_vjp(**changed):
    a = dict(grad_A=_array((7, 4)), grad_W=_array((9, 4)), grad_loss=_array((7,)), grad_log_sum=_array((7,)), loss=_array((7,)), log_sum=_array((7,)),
             A=_array((7, 4)), W=_array((9, 4)), targets=_t7, scale=1.0, ignore=-1)
    a.update(changed)
    return list(a.values())


@pytest.mark.parametrize("name,arguments,message", [
    ("grouped_gated_product", [_array((7, 3)), _array((7, 4)), _array((2, 4, 7)), _o3, 0], "an even number in all"),
    ("grouped_gated_product", [_array((7, 6)), _array((7, 4)), _array((2, 4, 6)), _o3, 0], "the sizes of one half of W along dimension 2 and output"),
    ("grouped_gated_product", [_array((7, 3)), _array((7, 4)), _array((2, 5, 6)), _o3, 0], "the sizes of W along dimension 1 and A along dimension 1"),
    ("grouped_gated_product", [_array((7, 3)), _array((7, 4)), _array((3, 4, 6)), _o3, 0], "and offsets along dimension 0 must match"),
    ("grouped_gated_product", [_array((7, 3)), _array((7, 4)), _array((2, 4, 6)), _o3, 2], "unknown activation 2 in cuda_grouped_gated_product"),
    ("grouped_gated_product", [_array((7, 3), stride=(4, 1)), _array((7, 4)), _array((2, 4, 6)), _o3, 0], "output must be contiguous"),
    ("grouped_gated_product", [_array((7, 3)), _array((7, 4)), _array((2, 4, 6), stride=(48, 12, 2)), _o3, 0], "W must have a stride of 1"),
    ("grouped_gated_product_vjp", [_array((7, 4)), _array((2, 4, 8)), _array((7, 3)), _array((7, 4)), _array((2, 4, 6)), _o3, 0],
     "the sizes of W along dimension 2 and grad_W along dimension 2"),
    ("grouped_gated_product_vjp", [_array((6, 4)), _array((2, 4, 6)), _array((7, 3)), _array((7, 4)), _array((2, 4, 6)), _o3, 0],
     "the sizes of A along dimension 0 and grad_A along dimension 0"),
    ("linear_cross_entropy", _loss(loss=_array((7,), "bfloat16")), "Expected loss to be of type float32"),
    ("linear_cross_entropy", _loss(A=_array((7, 4), "float64")), "Expected W to be of type float64"),
    ("linear_cross_entropy", _loss(W=_array((9, 5))), "the sizes of W along dimension 1 and A along dimension 1"),
    ("linear_cross_entropy", _loss(targets=_array((6,), "int32")), "the sizes of A along dimension 0 and targets along dimension 0"),
    ("linear_cross_entropy", _loss(log_sum=_array((8,))), "the sizes of A along dimension 0 and log_sum along dimension 0"),
    ("linear_cross_entropy", _loss(W=_array((0, 4))), "W must have a row"),
    ("linear_cross_entropy", _loss(scale=0.0), "scale must be positive and finite"),
    ("linear_cross_entropy", _loss(scale=float("nan")), "scale must be positive and finite"),
    ("linear_cross_entropy", _loss(scale=float("inf")), "scale must be positive and finite"),
    ("linear_cross_entropy", _loss(W=_array((9, 4), stride=(1, 9))), "W must have a last dimension of stride 1"),
    ("linear_cross_entropy", _loss(targets=_array((7,), "int32", (2,))), "targets must have a last dimension of stride 1"),
    ("linear_cross_entropy_vjp", _loss_vjp(grad_loss=_array((6,))), "and grad_loss along dimension 0 must match"),
    ("linear_cross_entropy_vjp", _loss_vjp(grad_log_sum=_array((7,), "float16")), "Expected grad_log_sum to be of type float32"),
    ("linear_cross_entropy_vjp", _loss_vjp(grad_W=_array((9, 3))), "the sizes of W along dimension 1 and grad_W along dimension 1"),
    ("linear_cross_entropy_vjp", _loss_vjp(grad_A=_array((7, 4), stride=(8, 1))), "grad_A must be contiguous"),
])
def test_entry_points_refuse_wrong_arrays(name, arguments, message):
    from mops_b200 import _lib
    integer = ctypes.c_int32 if "gated" in name else ctypes.c_int64
    scalar = [ctypes.c_double(a) if isinstance(a, float) else integer(a) if isinstance(a, int) else a for a in arguments]
    with pytest.raises(_lib.MopsError, match=message) as e:
        _lib.call(f"mops_b200_cuda_{name}", scalar)
    assert e.value.status == 1


@pytest.mark.parametrize("norm,outputs,gradients,max_norm,message", [
    (_array((1,), "float64", data=0x8000), None, [_array((5,))], 1.0, "Expected norm to be of type float32"),
    (_array((1,), data=0x8000), None, [_array((5,)), _array((5,), "float64")], 1.0, "Expected norm to be of type float64"),
    (_array((2,), data=0x8000), None, [_array((5,))], 1.0, "norm must have one value"),
    (_array((1,), data=0x8000), None, [_array((5,), "int32")], 1.0, "Wrong dtype for a gradient"),
    (_array((1,), data=0x8000), None, [_array((5, 4), stride=(8, 1))], 1.0, "a gradient must be contiguous"),
    (_array((1,), data=0x8000), [_array((4,), data=0x2000)], [_array((5,))], 1.0, "the sizes of its gradient along dimension 0 and an output"),
    (_array((1,), data=0x8000), [_array((5,), "bfloat16", data=0x2000)], [_array((5,))], 1.0, "Expected an output to be of type float32"),
    (_array((1,), data=0x8000), [_array((5,))], [_array((5,))], -1.0, "max_norm must not be negative"),
    (_array((1,), data=0x8000), [_array((5,))], [_array((5,))], float("nan"), "max_norm must not be negative"),
    (_array((1,), data=0x8000), [_array((5,))] * 2, [_array((5,))] * 2, 1.0, "gradients and outputs overlap"),
    (_array((1,), data=0x8000), [_array((5,), data=0x1004)], [_array((5,))], 1.0, "gradients and outputs overlap"),
    (_array((1,), data=0x2010), [_array((5,), data=0x2000)], [_array((5,))], 1.0, "gradients and outputs overlap"),
    (_array((1,), data=0x100c), None, [_array((5,))], 1.0, "gradients and norm overlap"),
    (_array((1,), data=0x8000), [_array((5,)), _array((5,), data=0x1010)], [_array((5,)), _array((5,), data=0x1010)], 1.0, "gradients and outputs overlap"),
])
def test_norm_refuses_wrong_arrays(norm, outputs, gradients, max_norm, message):
    from mops_b200 import _lib
    table = lambda arrays: (_lib.Array * len(arrays))(*arrays)
    n = ctypes.c_int64(len(gradients))
    with pytest.raises(_lib.MopsError, match=message):
        if outputs is None:
            _lib.call("mops_b200_cuda_gradient_norm", [norm, table(gradients), n])
        else:
            _lib.call("mops_b200_cuda_clip_gradient_norm", [norm, table(outputs), table(gradients), n, ctypes.c_double(max_norm)])


# ================================================================== grouped_gated_product
def gate(u, activation):
    if activation == "silu":
        s = torch.sigmoid(u)
        return u * s, s + u * s * (1 - s)
    phi = 0.5 * torch.erfc(-u / math.sqrt(2))
    return u * phi, phi + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)


def gated_plain(A, W, offsets, grad, activation):
    """Values and bounds of (output, grad_A, grad_W)."""
    u_, v_ = unit(A.dtype), inner_round(A.dtype)
    A, W, grad = A.double(), W.double(), grad.double()
    N, K = W.shape[2] // 2, A.shape[1]
    new = lambda *s: torch.zeros(*s, device=A.device, dtype=torch.float64)
    values, errors = ([new(A.shape[0], N), torch.zeros_like(A), torch.zeros_like(W)] for _ in range(2))
    bounds = offsets.tolist()
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        a, w, d = A[lo:hi], W[g], grad[lo:hi]
        uv, e = a @ w, 4 * (K + 4) * u_ * (a.abs() @ w.abs())
        (u, v), (eu, ev) = uv.chunk(2, 1), e.chunk(2, 1)
        f, slope = gate(u, activation)
        own = 32 * u_ * (1 + u.abs())
        values[0][lo:hi] = f * v
        errors[0][lo:hi] = (1.2 * eu + own) * (v.abs() + ev) + f.abs() * ev
        duv = torch.cat([d * v * slope, d * f], 1)
        eduv = torch.cat([d.abs() * ((slope.abs() + 1.2 * eu + own) * ev + v.abs() * (1.2 * eu + own)), d.abs() * (1.2 * eu + own)], 1)
        eduv += v_ * (duv.abs() + eduv) + (2.0 ** -25 if v_ == 2.0 ** -11 else 0)
        values[1][lo:hi], values[2][g] = duv @ w.T, a.T @ duv
        errors[1][lo:hi] = eduv @ w.abs().T + 4 * (2 * N + 4) * u_ * (duv.abs() @ w.abs().T)
        errors[2][g] = a.abs().T @ eduv + 4 * (hi - lo + 4) * u_ * (a.abs().T @ duv.abs())
    return values, errors


def check_gated(A, W, offsets, grad, activation="silu"):
    A, W = A.requires_grad_(True), W.requires_grad_(True)
    output = mt.grouped_gated_product(A, W, offsets, activation)
    got = [output.detach(), *torch.autograd.grad(output, [A, W], grad)]
    for g, w, e, what in zip(got, *gated_plain(A.detach(), W.detach(), offsets, grad, activation), ("output", "grad_A", "grad_W")):
        within(g, w, e, what)
    again = mt.grouped_gated_product(A, W, offsets, activation)
    assert torch.equal(again, output)
    for a, b in zip(torch.autograd.grad(again, [A, W], grad), got[1:]):
        assert torch.equal(a, b)
    assert torch.equal(mt.grouped_gated_product(A.detach(), W.detach(), offsets, activation), output)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K,N,activation", [
    ([1], 1, 1, "silu"), ([1], 64, 64, "gelu"), ([3, 0, 5], 7, 9, "gelu"), ([0, 0, 4, 0], 16, 24, "silu"), ([64, 64], 64, 128, "gelu"),
    ([63, 65, 1], 72, 136, "silu"), ([128, 129, 127], 128, 256, "gelu"), ([200, 0, 1, 300], 264, 40, "silu"), ([1] * 40, 32, 48, "silu"),
    ([17, 700], 96, 520, "gelu"), ([2000], 8, 16, "silu"), ([5, 1, 250], 509, 131, "silu"), ([33, 31], 1030, 30, "gelu"), ([0, 0], 16, 16, "silu"),
    ([1000, 1], 130, 258, "silu"), ([7] * 70, 16, 16, "gelu"), ([3000, 0, 129, 2500], 136, 500, "silu"), ([1111, 4000], 600, 385, "gelu"),
    ([30, 1, 33], 24, 33, "silu")])
def test_gated_matches_64_bits(dtype, rows, K, N, activation):
    R = sum(rows)
    check_gated(normal((R, K), dtype, 1), normal((len(rows), K, 2 * N), dtype, 2, 2 * K ** -0.5), offsets_of(rows), normal((R, N), dtype, 3), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("other_way", [False, True])
@pytest.mark.parametrize("before,rows,after,K,N", [
    (0, [1], 0, 4096, 8), (1, [0, 2, 0], 2, 1096, 1032), (0, [1] * 20 + [0] * 30 + [12], 0, 584, 136), (3, [17, 0, 1], 4, 264, 72),
    (0, [32], 0, 2048, 136), (0, [9, 70, 0, 20], 1, 1000, 264), (0, [2, 5, 1, 0, 3], 0, 1536, 512), (0, [0, 0, 0], 7, 128, 64),
    (0, [1, 2, 0, 1], 0, 35, 13)])
def test_gated_few_rows(dtype, other_way, before, rows, after, K, N):
    """Single tokens, rows of no group around them, and matrices stored either way round."""
    R = before + sum(rows) + after
    W = normal((len(rows), 2 * N, K), dtype, 2, K ** -0.5).transpose(1, 2) if other_way else normal((len(rows), K, 2 * N), dtype, 2, K ** -0.5)
    check_gated(normal((R, K), dtype, 1), W, offsets_of(rows) + before, normal((R, N), dtype, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(64, 128), (72, 40), (33, 65), (130, 300)])
def test_gated_matrices_stored_the_other_way(dtype, K, N):
    rows = [100, 0, 37, 260]
    W = normal((4, 2 * N, K), dtype, 4, K ** -0.5).transpose(1, 2)
    check_gated(normal((397, K), dtype, 5), W, offsets_of(rows), normal((397, N), dtype, 6), "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_on_strided_and_shifted_tensors(dtype):
    rows = [70, 3, 140]
    offsets = offsets_of(rows)
    A, W, grad = normal((213, 300), dtype, 7), normal((3, 160, 200), dtype, 8, 0.1), normal((213, 300), dtype, 9)
    for a, w, g in ((A[:, :128], W[:, :128, :96], grad[:, :48]), (A[:, 8:136], W[:, 8:136, 8:104], grad[:, 16:64]),
                    (A[:, 3:131], W[:, 1:129, 5:101], grad[:, 1:49]), (A[:, ::2][:, :64], W[:, :64:, ::2], grad[:, ::3][:, :50]),
                    (A[:, :128], W[:, :128, :96], grad[:1, :48].expand(213, 48)), (A[:, :128], W[:, :128, :96], grad[:, :1].expand(213, 48)),
                    (A[:, :128].T.contiguous().T, W[:, :128, 2:96], grad[:, :47])):
        check_gated(a.detach(), w.detach(), offsets, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [72, 35])
def test_gated_rows_of_no_group_and_empty_sizes(dtype, N):
    offsets = torch.tensor([5, 9, 9, 140], dtype=torch.int32, device="cuda")
    A, W, grad = normal((150, 64), dtype, 1), normal((3, 64, 2 * N), dtype, 2, 0.1), normal((150, N), dtype, 3)
    # what stands in rows of no group does not matter
    A[:5], A[140:], grad[:5], grad[140:] = float("nan"), float("inf"), float("nan"), float("-inf")
    A.requires_grad_(True), W.requires_grad_(True)
    output = mt.grouped_gated_product(A, W, offsets)
    gA, gW = torch.autograd.grad(output, [A, W], grad)
    for got, want, error in zip((output.detach(), gA, gW), *gated_plain(A.detach(), W.detach(), offsets, grad, "silu")):
        within(got, want, error)
    for t in (output[:5], output[140:], gA[:5], gA[140:], gW[1]):
        assert (t == 0).all()
    for R, G, K, n in ((0, 2, 4, 4), (6, 0, 4, 4), (6, 2, 0, 4), (6, 2, 4, 0), (100, 0, 8, 8), (100, 2, 0, 8), (100, 1, 8, 0)):
        o = torch.zeros(G + 1, dtype=torch.int32, device="cuda")
        if G:
            o[1:] = R
        a, w = normal((R, K), dtype, 1).requires_grad_(True), normal((G, K, 2 * n), dtype, 2).requires_grad_(True)
        out = mt.grouped_gated_product(a, w, o)
        assert out.shape == (R, n) and (out == 0).all()
        for x, like in zip(torch.autograd.grad(out, [a, w], torch.ones_like(out), allow_unused=True), (a, w)):
            assert x is None or (x.shape == like.shape and (x == 0).all())


@pytest.mark.gpu
def test_operators_refuse_what_does_not_fit():
    A, o = normal((70, 16), torch.bfloat16, 1), offsets_of([70])
    with pytest.raises(RuntimeError, match="an even number in all, in cuda_grouped_gated_product"):
        mt.grouped_gated_product(A, normal((1, 16, 7), torch.bfloat16, 2), o)
    with pytest.raises(RuntimeError, match="the sizes of W along dimension 1 and A along dimension 1 must match"):
        mt.grouped_gated_product(A, normal((1, 24, 8), torch.bfloat16, 2), o)
    with pytest.raises(RuntimeError, match="and offsets along dimension 0 must match"):
        mt.grouped_gated_product(A, normal((2, 16, 8), torch.bfloat16, 2), o)
    T, t = normal((9, 16), torch.bfloat16, 3), some_targets(70, 9, 1.0)
    with pytest.raises(RuntimeError, match="scale must be positive"):
        mt.linear_cross_entropy(A, T, t, -1.0)
    with pytest.raises(RuntimeError, match="W must have a row"):
        mt.linear_cross_entropy(A, T[:0], t)
    with pytest.raises(RuntimeError, match="the sizes of targets along dimension 0|and targets along dimension 0 must match"):
        mt.linear_cross_entropy(A, T, t[:-1])
    with pytest.raises(ValueError, match="All tensors must be on the same device"):
        mt.linear_cross_entropy(A, T, t.cpu())
    with pytest.raises(ValueError, match="All tensors must be on the same device"):
        mt.clip_gradient_norm([A, T.cpu()], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gated_reports_wrong_offsets(dtype):
    for R in (20, 300):
        A, W, grad = normal((R, 16), dtype, 1), normal((3, 16, 16), dtype, 2), normal((R, 8), dtype, 3)
        for bad in ([0, 5, 4, R], [-1, 5, 9, R], [0, 5, 9, R + 1], [0, 2 ** 31 - 1, 9, R]):
            offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
            with pytest.raises(mops_b200.MopsError, match="Index array offsets in operation cuda_grouped_gated_product"):
                mops_b200.grouped_gated_product(A, W, offsets)
            with pytest.raises(mops_b200.MopsError, match="Index array offsets in operation cuda_grouped_gated_product_vjp"):
                mops_b200.grouped_gated_product_vjp(grad, A, W, offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [30, 300])
def test_gated_nan_stays_in_its_rows(dtype, R):
    A, W, grad = normal((R, 64), dtype, 1), normal((2, 64, 96), dtype, 2, 0.1), normal((R, 48), dtype, 3)
    offsets = offsets_of([R // 2 - 2, R // 2 + 2])
    dirty, at = A.clone(), R // 2 - 3
    dirty[at] = float("nan")
    clean, got = (mops_b200.grouped_gated_product(a, W, offsets) for a in (A, dirty))
    rest = torch.arange(R, device="cuda") != at
    assert torch.equal(got[rest], clean[rest]) and got[at].isnan().all()
    (clean_A, clean_W), (got_A, got_W) = (mops_b200.grouped_gated_product_vjp(grad, a, W, offsets) for a in (A, dirty))
    assert torch.equal(got_A[rest], clean_A[rest]) and got_A[at].isnan().all()
    assert torch.equal(got_W[1], clean_W[1]) and got_W[0].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gated_far_from_zero(dtype, activation):
    """Gates that are closed or open all the way: no infinities on the way, and slopes of 0 and 1."""
    u = torch.tensor([-1e4, -200.0, -89.0, -30.0, -8.0, 0.0, 8.0, 30.0, 100.0, 1e4], device="cuda").to(dtype)
    R = 70
    A = torch.zeros(R, 8, dtype=dtype, device="cuda")
    A[:, 0], A[:, 1] = u.repeat(7), 1.0
    W = torch.zeros(1, 8, 16, dtype=dtype, device="cuda")
    W[0, 0, :8], W[0, 1, 8:] = 1.0, 2.0
    check_gated(A, W, offsets_of([R]), torch.ones(R, 8, dtype=dtype, device="cuda"), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_on_broadcast_tensors(dtype):
    """One matrix for all groups, one row for all rows, one gradient for all results: strides of zero."""
    offsets, one = offsets_of([100, 0, 150, 50]), torch.ones((), device="cuda", dtype=dtype)
    check_gated(normal((300, 64), dtype, 1), normal((1, 64, 96), dtype, 2, 0.125).expand(4, 64, 96), offsets, one.expand(300, 48))
    check_gated(normal((1, 64), dtype, 1).expand(300, 64), normal((4, 64, 96), dtype, 2, 0.125), offsets, normal((300, 48), dtype, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("other_way", [False, True])
@pytest.mark.parametrize("K,N", [(33, 65), (64, 96), (137, 261)])
def test_gated_matrices_of_empty_groups_are_not_read(dtype, other_way, K, N):
    rows = [0, 70, 0, 0, 400, 1, 0]
    W = normal((7, 2 * N, K) if other_way else (7, K, 2 * N), dtype, 2, K ** -0.5)
    W[[i for i, n in enumerate(rows) if n == 0]] = float("nan")
    check_gated(normal((471, K), dtype, 1), W.transpose(1, 2) if other_way else W, offsets_of(rows), normal((471, N), dtype, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [5, 3000])
def test_gated_of_more_groups_than_a_grid_is_wide(dtype, R):
    rows = torch.bincount(torch.randint(70000, (R,), generator=torch.Generator().manual_seed(1)), minlength=70000)
    A, W, grad = normal((R, 8), dtype, 1), normal((70000, 8, 16), dtype, 2, 0.35), normal((R, 8), dtype, 3)
    offsets = offsets_of(rows.tolist())
    full = rows.nonzero()[:, 0]
    A_, W_ = A.clone().requires_grad_(True), W.clone().requires_grad_(True)
    output = mt.grouped_gated_product(A_, W_, offsets)
    grad_A, grad_W = torch.autograd.grad(output, [A_, W_], grad)
    values, errors = gated_plain(A, W[full.cuda()], offsets_of(rows[full].tolist()), grad, "silu")
    for g, w, e, what in zip((output.detach(), grad_A, grad_W[full.cuda()]), values, errors, ("output", "grad_A", "grad_W")):
        within(g, w, e, what)
    grad_W[full.cuda()] = 0
    assert (grad_W == 0).all()


# ================================================================== linear_cross_entropy
def loss_plain(A, W, targets, scale, ignored, grad_loss, grad_log_sum):
    """Values and bounds of (loss, log_sum, grad_A, grad_W)."""
    u_, v_ = unit(A.dtype), inner_round(A.dtype)
    # What is lost of an operand of the products whatever its size: f16 below its smallest value, as they are scaled to the largest gradient; bf16 and f32 below
    # the smallest that is kept in three parts (2^-133) or comes out of an exponential (2^-126, times the gradient); f64 below 2^-1074.
    small = {torch.float16: 2.0 ** -36, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126, torch.float64: 2.0 ** -1074}[A.dtype]
    keep = targets != ignored
    t = torch.where(keep, targets, 0).long()
    A, W = torch.where(keep[:, None], A.double(), 0.0), W.double()
    V, C = W.shape
    x = scale * (A @ W.T)
    ex = scale * 4 * (C + 4) * u_ * (A.abs() @ W.abs().T) + 4 * u_ * x.abs()
    log_sum = torch.logsumexp(x, 1)
    x_t = x.gather(1, t[:, None])[:, 0]
    e_sum = ex.amax(1) + (400 + V / 64) * u_ + 4 * u_ * log_sum.abs()
    e_loss = e_sum + ex.gather(1, t[:, None])[:, 0] + 4 * u_ * (log_sum.abs() + x_t.abs())
    gl, gs = (torch.where(keep, g.double(), 0.0)[:, None] for g in (grad_loss, grad_log_sum))
    p = torch.exp(x - log_sum[:, None])
    dx = (gl + gs) * p
    # the exponent's own rounding, too
    e_dx = dx.abs() * (ex + e_sum[:, None] + 32 * u_ * (1 + (x - log_sum[:, None]).abs()))
    # (at the target p is also exp(-loss), which is off as the loss is)
    e_dx.scatter_add_(1, t[:, None], (dx.gather(1, t[:, None]).abs() * 2 * e_loss[:, None] + 4 * u_ * gl.abs()))
    dx.scatter_add_(1, t[:, None], -gl)
    e_dx += v_ * (dx.abs() + e_dx) + small * (1 + (gl.abs() + gs.abs()).max())
    e_dx *= keep[:, None]
    values = [torch.where(keep, log_sum - x_t, 0.0), torch.where(keep, log_sum, 0.0), scale * dx @ W, scale * dx.T @ A]
    errors = [keep * e_loss, keep * e_sum, scale * (e_dx @ W.abs() + 4 * (V + 4) * u_ * (dx.abs() @ W.abs())),
              scale * (e_dx.T @ A.abs() + 4 * (A.shape[0] + 4) * u_ * (dx.abs().T @ A.abs()))]
    return values, errors


def check_loss(A, W, targets, scale=1.0, ignored=-1, seed=9, weights=None):
    A, W = A.requires_grad_(True), W.requires_grad_(True)
    sums = torch.float64 if A.dtype == torch.float64 else torch.float32
    grad_loss, grad_log_sum = (normal((A.shape[0],), sums, seed + i) for i in range(2))
    if weights is not None:
        grad_loss, grad_log_sum = weights
    outputs = mt.linear_cross_entropy(A, W, targets, scale, ignored)
    got = [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, [A, W], [grad_loss, grad_log_sum]))
    assert got[0].dtype == sums and got[1].dtype == sums
    values, errors = loss_plain(A.detach(), W.detach(), targets, scale, ignored, grad_loss, grad_log_sum)
    for g, w, e, what in zip(got, values, errors, ("loss", "log_sum", "grad_A", "grad_W")):
        within(g, w, e, what)
    ignored_rows = targets == ignored
    assert (got[0][ignored_rows] == 0).all() and (got[1][ignored_rows] == 0).all() and (got[2][ignored_rows] == 0).all()
    again = mt.linear_cross_entropy(A, W, targets, scale, ignored)
    for a, b in zip(list(again) + list(torch.autograd.grad(again, [A, W], [grad_loss, grad_log_sum])), got):
        assert torch.equal(a, b)
    for a, b in zip(mt.linear_cross_entropy(A.detach(), W.detach(), targets, scale, ignored), got):
        assert torch.equal(a, b)
    return got


def some_targets(R, V, kept, seed=5, ignored=-1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(V, (R,), generator=gen, device="cuda")
    return torch.where(torch.rand(R, generator=gen, device="cuda") < kept, t, ignored).to(torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C,kept", [
    (1, 1, 1, 1.0), (1, 2, 8, 1.0), (2, 5, 3, 1.0), (1, 5000, 64, 1.0), (3, 257, 40, 0.5), (8, 1000, 1030, 1.0), (31, 4097, 72, 0.8), (64, 63, 16, 1.0),
    (130, 300, 64, 0.9), (257, 1000, 129, 0.5), (300, 8200, 96, 0.95), (400, 129, 256, 0.7), (700, 5003, 203, 0.3), (1025, 2, 40, 0.9),
    (2000, 77, 520, 1.0), (513, 12345, 8, 0.9), (2049, 3000, 64, 0.9), (4100, 511, 72, 0.4), (300, 70001, 24, 0.9), (3000, 50001, 16, 0.9), (70000, 40, 8, 0.6), (9000, 3, 24, 0.5), (1100, 9001, 520, 0.8),
    (4224, 8191, 130, 0.94), (770, 12000, 1030, 1.0), (300, 100, 1, 1.0), (5000, 600, 136, 0.02), (385, 3000, 700, 0.99)])
def test_loss_matches_64_bits(dtype, R, V, C, kept):
    A, W = normal((R, C), dtype, 1, 2.0), normal((V, C), dtype, 2, C ** -0.5)
    check_loss(A, W, some_targets(R, V, kept), 1.25)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_of_a_mean(dtype):
    """Gradients that are the same for all rows, as of a mean, and many orders below one (f16: below its smallest value)."""
    R, V, C = 600, 3001, 200
    A, W, targets = normal((R, C), dtype, 1), normal((V, C), dtype, 2, C ** -0.5), some_targets(R, V, 0.9)
    sums = torch.float64 if dtype == torch.float64 else torch.float32
    for size in (1.0 / 541, 1e-12, 65536.0):
        even = torch.full((R,), size, dtype=sums, device="cuda")
        if dtype == torch.float16 and size < 1e-6:
            continue  # (their gradients are below it, too)
        check_loss(A.detach(), W.detach(), targets, weights=(even, torch.zeros_like(even)))
        check_loss(A.detach(), W.detach(), targets, weights=(even, even * 1e-4))
        check_loss(A.detach(), W.detach(), targets, weights=(torch.zeros_like(even), even))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C", [(20, 500, 72), (400, 500, 72), (1100, 9001, 520)])
def test_loss_rows_without_target(dtype, R, V, C):
    """What stands in rows without a target does not matter; all rows may be without one."""
    A, W, targets = normal((R, C), dtype, 1), normal((V, C), dtype, 2, 0.1), some_targets(R, V, 0.5, ignored=499)
    A[targets == 499] = float("nan")
    got = check_loss(A, W, targets, ignored=499)
    assert all(t.isfinite().all() for t in got)
    none = torch.full_like(targets, -7)
    a, w = A.detach().requires_grad_(True), W.detach().requires_grad_(True)
    loss, log_sum = mt.linear_cross_entropy(a, w, none, 1.0, -7)
    gA, gW = torch.autograd.grad(loss.sum() + log_sum.sum(), [a, w])
    for t in (loss, log_sum, gA, gW):
        assert (t == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [20, 400])
def test_loss_reports_targets_out_of_range(dtype, R):
    V, C = 300, 64
    A, W, targets = normal((R, C), dtype, 1), normal((V, C), dtype, 2, 0.1), some_targets(R, V, 0.9)
    want = check_loss(A.detach(), W.detach(), targets.clone().index_fill_(0, torch.tensor([3, 7, 11], device="cuda"), -1))
    bad = targets.clone()
    bad[3], bad[7], bad[11] = V, -2, 2 ** 31 - 1
    loss, log_sum = mt.linear_cross_entropy(A, W, bad)  # not waited for: rows of zeros
    assert torch.equal(loss, want[0]) and torch.equal(log_sum, want[1])
    with pytest.raises(mops_b200.MopsError, match="Index array targets in operation cuda_linear_cross_entropy contains"):
        mops_b200.linear_cross_entropy(A.detach(), W.detach(), bad)
    with pytest.raises(mops_b200.MopsError, match="Index array targets in operation cuda_linear_cross_entropy_vjp contains"):
        mops_b200.linear_cross_entropy_vjp(loss.detach(), None, loss.detach(), log_sum.detach(), A.detach(), W.detach(), bad)
    mops_b200.linear_cross_entropy(A.detach(), W.detach(), targets)  # the next call is not affected


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [30, 300])
def test_loss_on_strided_and_shifted_tensors(dtype, R):
    A, W = normal((R, 300), dtype, 1), normal((1000, 300), dtype, 2, 0.1)
    t = some_targets(2 * R, 400, 0.9)
    for a, w, targets in ((A[:, :128], W[:400, :128], t[:R]), (A[:, 8:136], W[100:500, 16:144], t[::2]), (A[:, 3:131], W[:800:2, 5:133], t[1:R + 1]),
                          (A[:, ::2], W[:400, ::2], t[:R]), (A[:1, :128].expand(R, 128), W[:400, :128], t[:R]),
                          (A[:, :128].T.contiguous().T, W[:400, :128].T.contiguous().T, t[:R]), (A[:, :128], W[:1, :128].expand(400, 128), t[:R])):
        check_loss(a.detach(), w.detach(), targets)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C,stride", [
    (1, 1, 8, 8), (1, 7, 8, 8), (3, 15, 24, 40), (8, 16, 32, 32), (9, 17, 37, 40), (16, 2400, 40, 40), (17, 2400, 40, 40), (8, 100, 1000, 1000), (7, 3001, 2064, 2064),
    (16, 50021, 64, 64), (5, 40000, 255, 256), (6, 900, 37, 37), (12, 5000, 146, 146), (16, 130, 2050, 2050), (16, 300, 3200, 3200), (3, 200, 6500, 6501)])
def test_loss_of_few_rows(dtype, R, V, C, stride):
    table = normal((V, stride), dtype, 2, C ** -0.5)
    table[:, C:] = float("nan")
    targets = torch.tensor([V - 1, 0, -1, V // 2], device="cuda", dtype=torch.int32)[torch.arange(R, device="cuda") % 4]
    check_loss(normal((R, C), dtype, 1, 2.0), table[:, :C], targets, 1.5)
    assert not mt.linear_cross_entropy(normal((R, C), dtype, 1), table[:, :C], targets)[0].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [200, 3000])
def test_loss_after_one_of_nan(dtype, R):
    """What a call leaves in workspaces is not found again: rows behind the last one that counts are zeros there."""
    A, W = normal((R, 264), dtype, 1), normal((6000, 264), dtype, 2, 0.125)
    leaves = [torch.full_like(A, float("nan")).requires_grad_(True), W.clone().requires_grad_(True)]
    loss = mt.linear_cross_entropy(*leaves, some_targets(R, 6000, 1.0))[0]
    assert loss.isnan().all() and torch.autograd.grad(loss.sum(), leaves)[1].isnan().all()
    check_loss(A, W, some_targets(R, 6000, 0.37))
    check_loss(A.detach(), W.detach(), torch.arange(R, dtype=torch.int32, device="cuda") % 7, ignored=5)
    check_loss(A.detach(), W.detach(), torch.full((R,), 5, dtype=torch.int32, device="cuda"), ignored=5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C", [(130, 7, 2049), (674, 61, 2600), (40, 1999, 2300), (1, 3, 2500)])
def test_loss_of_few_tiles_of_much_depth(dtype, R, V, C):
    """Also where an operand is infinite, and rows and table begin anywhere."""
    A, W = normal((R, C + 3), dtype, 1)[:, 1:C + 1], normal((V, C + 1), dtype, 2, C ** -0.5)[:, 1:]
    targets = some_targets(R, V, 0.8)
    check_loss(A, W, targets, 1.25)
    A = A.detach().clone()
    A[R // 2, C - 1] = float("inf")
    targets[R // 2] = 0
    loss, log_sum = mt.linear_cross_entropy(A, W.detach(), targets)
    assert not log_sum[R // 2].isfinite() and log_sum.isfinite().sum() == R - 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_of_many_logits_on_strided_tensors(dtype):
    A, W, t = normal((900, 1300), dtype, 1), normal((9100, 1300), dtype, 2, 0.1), some_targets(900, 9000, 0.9)
    for a, w in ((A[:, :516], W[:9000, 4:520]), (A[:, 3:523], W[100:9100, 5:525]), (A[:, ::2], W[:9000, ::2]), (A[:1, :512].expand(900, 512), W[:9000, :512])):
        check_loss(a.detach(), w.detach(), t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_of_many_rows_is_that_of_each(dtype):
    """So many rows that they are taken in turns: each has the loss that it has among a few."""
    R, V, C = 70000, 150001, 8
    A, W, t = normal((R, C), dtype, 1), normal((V, C), dtype, 2, 0.3), some_targets(R, V, 0.9)
    loss, log_sum = mt.linear_cross_entropy(A, W, t)
    for rows in (slice(0, 40), slice(56000, 57600), slice(R - 300, R)):
        values, errors = loss_plain(A[rows], W, t[rows], 1.0, -1, *(torch.ones(R, device="cuda")[rows] for _ in range(2)))
        within(loss[rows], values[0], errors[0], "loss")
        within(log_sum[rows], values[1], errors[1], "log_sum")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,C", [(9, 700, 16), (300, 700, 16), (600, 13001, 520)])
def test_loss_of_large_and_infinite_logits(dtype, R, V, C):
    A, W = normal((R, C), dtype, 1, 100.0), normal((V, C), dtype, 2, 10.0)
    targets = some_targets(R, V, 1.0)
    check_loss(A, W, targets)  # most p are zero, some losses in the thousands
    clean = mt.linear_cross_entropy(A.detach(), W.detach(), targets)
    dirty = A.detach().clone()
    dirty[2] = float("nan")
    got = mt.linear_cross_entropy(dirty, W.detach(), targets)
    rest = torch.arange(R, device="cuda") != 2
    for g, c in zip(got, clean):
        assert torch.equal(g[rest], c[rest]) and g[2].isnan()
    # one column that is infinite for positive first values, and -infinite for negative ones
    w = torch.zeros(V, C, dtype=dtype, device="cuda")
    w[5, 0] = float("inf")
    a = torch.ones(R, C, dtype=dtype, device="cuda")
    a[1::2, 0] = -1.0
    targets = torch.where(torch.arange(R, device="cuda") % 4 < 2, 6, 5).to(torch.int32)
    loss, log_sum = mt.linear_cross_entropy(a, w, targets)
    assert (log_sum[0::2] == float("inf")).all() and (loss[0::4] == float("inf")).all()
    assert (log_sum[1::2] - math.log(V - 1)).abs().max() < 1e-5
    assert (loss[1::4] - math.log(V - 1)).abs().max() < 1e-5 and (loss[3::4] == float("inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [9, 300, 2100])
@pytest.mark.parametrize("far", [-4.0, 4.0])
def test_loss_of_logits_far_from_zero(dtype, R, far):
    """All logits beyond what exponentials can be taken of, to either side."""
    V, C = 1300, 16
    A, W = 5 + normal((R, C), dtype, 1, 0.01), far + normal((V, C), dtype, 2, 0.05)
    check_loss(A, W, some_targets(R, V, 0.9))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_of_empty_sizes(dtype):
    W = normal((50, 24), dtype, 1).requires_grad_(True)
    A = normal((0, 24), dtype, 2).requires_grad_(True)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    loss, log_sum = mt.linear_cross_entropy(A, W, none)
    assert loss.shape == (0,) and log_sum.shape == (0,)
    gA, gW = torch.autograd.grad(loss.sum() + log_sum.sum(), [A, W])
    assert gA.shape == A.shape and (gW == 0).all()
    for R in (5, 300):  # logits of nothing are zero
        a, w = (normal((n, 0), dtype, 3).requires_grad_(True) for n in (R, 50))
        loss, log_sum = mt.linear_cross_entropy(a, w, some_targets(R, 50, 1.0))
        assert (loss - math.log(50)).abs().max() < 1e-5 and (log_sum - math.log(50)).abs().max() < 1e-5
        gA, gW = torch.autograd.grad(loss.sum(), [a, w])
        assert gA.shape == a.shape and gW.shape == w.shape


@pytest.mark.gpu
def test_loss_gradients_of_one_result_alone():
    for dtype, R in ((torch.float32, 40), (torch.bfloat16, 40), (torch.bfloat16, 300)):
        A, W, t = normal((R, 64), dtype, 1).requires_grad_(True), normal((90, 64), dtype, 2, 0.1).requires_grad_(True), some_targets(R, 90, 0.9)
        zero, g = torch.zeros(R, device="cuda"), normal((R,), torch.float32, 4)
        outputs = mt.linear_cross_entropy(A, W, t)
        for i in range(2):
            one = torch.autograd.grad(outputs[i], [A, W], g, retain_graph=True)
            both = torch.autograd.grad(outputs, [A, W], [g, zero] if i == 0 else [zero, g], retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(one, both))


# ======================================================================= norm of gradients
# Squares are off by u, sums of a thread's (at most 16 in f32, then f64) by 16 u, the root by half of it and its rounding by u: 10 u;
# the factor and its product by 2 u more.
NORM_ERROR = 10 * 2.0 ** -24


def check_clip(tensors, max_norm, finite=True):
    values = [t.double() for t in tensors]
    norm = math.sqrt(math.fsum(float((v * v).sum()) for v in values))
    factor = max_norm / norm if norm > max_norm else 1.0
    for result, clipped in (mt.clip_gradient_norm(tensors, max_norm), (mt.gradient_norm(tensors), None)):
        assert result.shape == () and abs(float(result) - norm) <= norm * NORM_ERROR + 1e-44
        if clipped is None:
            continue
        for c, v, t in zip(clipped, values, tensors):
            if factor == 1.0:
                assert torch.equal(c, t)
            else:
                within(c, v * factor, v.abs() * factor * (NORM_ERROR + 2 * 2.0 ** -24), "clipped")
    again = mt.clip_gradient_norm(tensors, max_norm)
    in_place = [t.clone() for t in tensors]
    versions = [t._version for t in in_place]
    assert torch.equal(mt.clip_gradient_norm_(in_place, max_norm), again[0])
    for a, b in zip(in_place, again[1]):
        assert torch.equal(a, b)
    assert all(t._version > v for t, v in zip(in_place, versions))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shapes", [[(1,)], [(3,), ()], [(0,), (5, 0), (7,)], [(1000,), (33, 17), (2, 3, 4)], [(40000,), (16384,), (8192, 3)], [(1,)] * 40,
                                    [(129, 257)] * 33, [(5,)] * 1000, [(3000001,), (7, 5, 11, 13)]])
@pytest.mark.parametrize("max_norm", [0.01, 1e9])
def test_norm_matches_64_bits(dtype, shapes, max_norm):
    check_clip([normal(s, dtype, i, 1.0 + i % 5) for i, s in enumerate(shapes)], max_norm)


@pytest.mark.gpu
def test_norm_of_several_types_and_places():
    base = [normal((70001,), d, 7 + i) for i, d in enumerate(DTYPES)]
    for cut in range(9):
        tensors = [b[cut:cut + 20000 + 3 * cut] for b in base] + [normal((cut, 5), torch.float32, 3), normal((64, 40), torch.bfloat16, 5).T]
        check_clip(tensors, 1.0)
        check_clip(tensors[:1] + tensors[2:], 1.0)  # (without f64)
    # gaps between rows: copies out of place, refused in place
    wide = normal((50, 60), torch.float32, 9)
    norm, (clipped,) = mt.clip_gradient_norm([wide[:, :30]], 1.0)
    within(clipped, wide[:, :30].double() / wide[:, :30].double().norm(), 1e-6)
    with pytest.raises(ValueError, match="without gaps"):
        mt.clip_gradient_norm_([wide[:, :30]], 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        mt.clip_gradient_norm_([wide, wide], 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        mt.clip_gradient_norm_([wide, wide[3]], 1.0)
    both = float(mt.gradient_norm([wide, wide]))  # (counted twice)
    assert abs(both - math.sqrt(2) * float(wide.double().norm())) < 1e-5 * both
    assert not torch.equal(mt.clip_gradient_norm([wide[:25], wide[25:]], 1.0)[1][0], wide[:25])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_that_is_zero_or_not_finite(dtype):
    zeros = [torch.zeros(300, dtype=dtype, device="cuda"), torch.zeros(7, dtype=dtype, device="cuda")]
    for max_norm in (0.0, 1.0):
        check_clip(zeros, max_norm)
    tensors = [normal((300,), dtype, 1), normal((5,), dtype, 2)]
    check_clip(tensors, 0.0)
    assert all((c == 0).all() for c in mt.clip_gradient_norm(tensors, 0.0)[1])
    for bad in (float("inf"), float("-inf"), float("nan")):
        tensors[1][3] = bad
        norm, clipped = mt.clip_gradient_norm(tensors, 1.0)
        assert not norm.isfinite() and norm.isnan() == math.isnan(bad)
        assert torch.equal(clipped[0], tensors[0]) and torch.equal(clipped[1].nan_to_num(), tensors[1].nan_to_num())
        kept = [t.clone() for t in tensors]
        mt.clip_gradient_norm_(kept, 1.0)
        assert torch.equal(kept[0], tensors[0])
    with pytest.raises(RuntimeError, match="max_norm must not be negative"):
        mt.clip_gradient_norm(tensors, -1.0)
    assert torch.equal(mt.clip_gradient_norm(tensors[:1], float("inf"))[1][0], tensors[0])


# ============================================================ what they have in common
def small_problems(dtype=torch.float64):
    offsets = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda")
    targets = torch.tensor([3, 0, -1, 6, 3], dtype=torch.int32, device="cuda")
    A, W, T = normal((5, 3), dtype, 1), normal((3, 3, 8), dtype, 2), normal((7, 3), dtype, 3)
    return [
        (lambda A, W: mt.grouped_gated_product(A, W, offsets, "silu"), [A, W]),
        (lambda A, W: mt.grouped_gated_product(A, W, offsets, "gelu"), [A, W]),
        (lambda A, T: mt.linear_cross_entropy(A, T, targets, 0.7), [A, T]),
    ]


@pytest.mark.gpu
def test_gradients_match_differences():
    for f, leaves in small_problems():
        assert torch.autograd.gradcheck(f, [t.clone().requires_grad_(True) for t in leaves])


@pytest.mark.gpu
def test_only_the_gradients_that_are_asked_for():
    for f, leaves in small_problems():
        full = [t.clone().requires_grad_(True) for t in leaves]
        out = f(*full)
        out = out if isinstance(out, tuple) else (out,)
        want = torch.autograd.grad(out, full, [torch.ones_like(t) for t in out])
        for i in range(len(leaves)):
            some = [t.clone().requires_grad_(j == i) for j, t in enumerate(leaves)]
            out = f(*some)
            out = out if isinstance(out, tuple) else (out,)
            got, = torch.autograd.grad(out, [some[i]], [torch.ones_like(t) for t in out])
            assert torch.equal(got, want[i])


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    for f, leaves in small_problems():
        leaves = [t.clone().requires_grad_(True) for t in leaves]
        out = f(*leaves)
        out = out[0] if isinstance(out, tuple) else out
        first = torch.autograd.grad(out.pow(2).sum(), leaves[:1], create_graph=True)[0]
        with pytest.raises(Exception, match="second derivatives are not supported"):
            first.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("R", [40, 600])
def test_a_step_on_other_streams_and_in_a_graph(R):
    """The operators together, as a training step has them: table, gated layer, product back, loss over the table, clipping. On the default
    stream, on another one than the tensors were made on, and captured and replayed on new values."""
    dtype, V, C, N = torch.bfloat16, 1000, 64, 96
    table, W1, W2 = normal((V, C), dtype, 1), normal((3, C, 2 * N), dtype, 2, C ** -0.5), normal((3, N, C), dtype, 3, N ** -0.5)
    offsets = offsets_of([R // 4, 0, R - R // 4])
    tokens, targets = some_targets(R, V, 1.0), some_targets(R, V, 0.9, 6)
    even = torch.full((R,), 1.0 / R, device="cuda")

    def step():
        rows = mops_b200.torch.embedding_lookup(table, tokens)
        h = mt.grouped_gated_product(rows, W1, offsets)
        out = mt.grouped_matrix_product(h, W2, offsets)
        loss, log_sum = mt.linear_cross_entropy(out, table, targets)
        # (gradients through the library's own entry points: nothing of autograd outlives the step)
        g_out, g_table = torch.empty_like(out), torch.empty_like(table)
        g_h, g_W2, g_rows, g_W1 = (torch.empty_like(t) for t in (h, W2, rows, W1))
        from mops_b200 import _lib
        lib = _lib.library()
        stream, waits = lib.mops_b200_get_stream(), lib.mops_b200_get_wait()
        lib.mops_b200_set_stream(torch.cuda.current_stream().cuda_stream)
        lib.mops_b200_set_wait(0)
        try:
            a = library_array
            _lib.call("mops_b200_cuda_linear_cross_entropy_vjp", [a(g_out), a(g_table), a(even), _lib.Array(), a(loss), a(log_sum), a(out), a(table), a(targets),
                                                                  ctypes.c_double(1.0), ctypes.c_int64(-1)])
            _lib.call("mops_b200_cuda_grouped_matrix_product_vjp", [a(g_h), a(g_W2), a(g_out), a(h), a(W2), a(offsets)])
            _lib.call("mops_b200_cuda_grouped_gated_product_vjp", [a(g_rows), a(g_W1), a(g_h), a(rows), a(W1), a(offsets), ctypes.c_int32(0)])
        finally:
            lib.mops_b200_set_stream(stream)
            lib.mops_b200_set_wait(waits)
        norm, clipped = mt.clip_gradient_norm([g_table, g_W1, g_W2], 1e-3)
        return [loss, log_sum, g_rows, norm, *clipped]

    want = [t.clone() for t in step()]
    leaves = [t.detach().requires_grad_(True) for t in (table, W1, W2)]
    out = mt.grouped_matrix_product(mt.grouped_gated_product(mt.embedding_lookup(table, tokens), leaves[1], offsets), leaves[2], offsets)
    recorded = torch.autograd.grad(mt.linear_cross_entropy(out, leaves[0], targets)[0], leaves, even)
    for g, w in zip(mt.clip_gradient_norm(recorded, 1e-3)[1], want[4:]):
        assert torch.equal(g, w)
    del leaves, out, recorded
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs, captured = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(step())
        graphs.append(graph)
    table.mul_(1.25)
    targets.copy_(some_targets(R, V, 0.8, 8))
    for graph in graphs + graphs[:1]:
        graph.replay()
    fresh = step()
    for c in captured:
        assert all(torch.equal(x, y) for x, y in zip(c, fresh))
    assert not torch.equal(fresh[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_with_autograd_in_a_graph(dtype):
    """Forward, gradients through autograd and clipping, captured after an eager step of which nothing is left, and replayed on new values."""
    leaves = [normal((1000, 64), dtype, 1), normal((3, 64, 192), dtype, 2, 0.125), normal((3, 96, 64), dtype, 3, 0.125)]
    leaves = [t.requires_grad_(True) for t in leaves]
    offsets, tokens, targets = offsets_of([100, 0, 500]), some_targets(600, 1000, 1.0), some_targets(600, 1000, 0.9, 6)

    def step():
        table, W1, W2 = leaves
        out = mt.grouped_matrix_product(mt.grouped_gated_product(mt.embedding_lookup(table, tokens), W1, offsets), W2, offsets)
        loss, log_sum = mt.linear_cross_entropy(out, table, targets)
        gradients = torch.autograd.grad(loss.mean() + 1e-3 * log_sum.mean(), leaves)
        norm, clipped = mt.clip_gradient_norm(gradients, 1e-3)
        return [loss.detach(), norm, *clipped]

    before = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        leaves[0].mul_(1.25)
    targets.copy_(some_targets(600, 1000, 0.8, 8))
    graph.replay()
    graph.replay()
    for c, f, b in zip(captured, step(), before):
        assert torch.equal(c, f) and not torch.equal(c, b)


@pytest.mark.gpu
def test_graphs_at_the_same_time():
    """Two captured steps, replayed over and over on two streams, have workspaces of their own."""
    def step(seed):
        A, W, t = normal((2000, 128), torch.bfloat16, seed), normal((9000, 128), torch.bfloat16, seed + 1, 0.1), some_targets(2000, 9000, 0.7, seed)
        M, offsets = normal((3, 128, 256), torch.bfloat16, seed + 2, 0.1), offsets_of([700, 600, 700])
        return lambda: [*mt.linear_cross_entropy(A, W, t), mt.grouped_gated_product(A, M, offsets), *mt.clip_gradient_norm([A, W], 0.1)[1]]

    steps = [step(11), step(23)]
    want = [[x.clone() for x in f()] for f in steps]
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in steps]
    for f in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(f())
        graphs.append(graph)
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))


@pytest.mark.gpu
def test_calls_from_several_threads():
    failures = []

    def work(seed, dtype):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3):
                    check_loss(normal((600 + seed, 72), dtype, seed), normal((900, 72), dtype, 2 + seed, 0.125), some_targets(600 + seed, 900, 0.7, seed))
                    check_gated(normal((500 + seed, 72), dtype, seed), normal((2, 72, 80), dtype, 2, 0.125), offsets_of([200, 300]), normal((500 + seed, 40), dtype, 9))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i, DTYPES[i % len(DTYPES)])) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]


@pytest.mark.gpu
def test_front_end_on_tensors_and_host_arrays():
    A, offsets = normal((40, 24), torch.float32, 2), offsets_of([10, 30])
    M, grad, T, t = normal((2, 24, 32), torch.float32, 3), normal((40, 16), torch.float32, 4), normal((30, 24), torch.float32, 5), some_targets(40, 30, 0.9)
    loss, log_sum = mops_b200.linear_cross_entropy(A, T, t.long(), 0.5)
    g = normal((40,), torch.float32, 6)
    calls = [
        (mops_b200.grouped_gated_product, [A, M, offsets, "gelu"]),
        (mops_b200.grouped_gated_product_vjp, [grad, A, M, offsets]),
        (mops_b200.linear_cross_entropy, [A, T, t, 0.5]),
        (mops_b200.linear_cross_entropy_vjp, [g, g, loss, log_sum, A, T, t, 0.5]),
    ]
    on_host = lambda x: x.cpu().numpy() if isinstance(x, torch.Tensor) else x
    for f, arguments in calls:
        want = f(*arguments)
        host = f(*[on_host(x) for x in arguments])
        with mops_b200.HostQueue():
            queued = f(*[on_host(x) for x in arguments])
        single = not isinstance(want, tuple)
        for w, h, q in zip(*([x] if single else x for x in (want, host, queued))):
            assert isinstance(h, np.ndarray) and np.array_equal(w.cpu().numpy(), h) and np.array_equal(h, q)
    assert mops_b200.grouped_gated_product_vjp(grad, A, M, offsets, compute_grad_W=False)[1] is None
    assert mops_b200.linear_cross_entropy_vjp(g, None, loss, log_sum, A, T, t, 0.5, compute_grad_A=False)[0] is None
    half = mops_b200.linear_cross_entropy(A.half(), T.half(), t)
    assert half[0].dtype == torch.float32
    tensors = [A, M.double(), grad.half()]
    norm, clipped = mops_b200.clip_gradient_norm(tensors, 2.0)
    host = [on_host(x) for x in tensors]
    host_norm, host_clipped = mops_b200.clip_gradient_norm(host, 2.0)
    with mops_b200.HostQueue():
        queued_norm, queued = mops_b200.clip_gradient_norm(host, 2.0)
    assert float(norm) == float(host_norm) == float(queued_norm) == float(mops_b200.gradient_norm(host))
    for c, h, q in zip(clipped, host_clipped, queued):
        assert h.dtype == on_host(c).dtype and np.array_equal(on_host(c), h) and np.array_equal(h, q)
