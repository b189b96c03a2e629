"""The operators of the block (embedding_lookup, grouped_matrix_product, gated_residual_norm): refusals on the CPU; on
the GPU, forward and gradients against a plain implementation in 64 bits, and gradients against differences.

Tolerances. Every output is a sum held in 32 bits (f64: 64) of n products of operands that are exact in the
given type, rounded once at the end: with u the unit roundoff of the sum's type and v that of the output's, the error of
one value is at most v |value| + n u sum|terms| to first order. u = 2^-24 (2^-53 for f64), v = 2^-11 (f16), 2^-8
(bf16), 2^-24 (f32), 2^-53 (f64). The bounds are taken value by value. For f32 products on tensor cores every factor is
split into parts that carry 24 bits, and sums are truncated where they would be rounded: four times the bound of the sum
covers both. Each test computes sum|terms| with the same plain code on absolute values.
"""
import numpy as np
import pytest
import torch

import mops_b200
import mops_b200.torch as mt

DTYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
ROUND = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SUM = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -24}
SMALLEST = {torch.float32: 1e-44, torch.float64: 1e-320, torch.float16: 6e-8, torch.bfloat16: 1e-40}


def close(got, want, terms, n, what=""):
    """Value by value: |got - want| <= v |want| + 4 n u terms (terms: the sums of absolute values)."""
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    error = (got.double() - want).abs()
    bound = ROUND[got.dtype] * want.abs() + 4 * (n + 4) * SUM[got.dtype] * terms + SMALLEST[got.dtype]
    worst = (error - bound).max().item() if error.numel() else 0.0
    assert not (error > bound).any() and not error.isnan().any(), f"{what}: over the bound by {worst:.3e}"


def normal(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64) * scale).to(dtype)


# =============================================================================== refusals
def test_schemas():
    schemas = {
        "embedding_lookup":
            "mops::embedding_lookup(Tensor W, Tensor indices, float scale=1., int padding_index=-1) -> Tensor",
        "grouped_matrix_product": "mops::grouped_matrix_product(Tensor A, Tensor W, Tensor offsets) -> Tensor",
        "gated_residual_norm":
            "mops::gated_residual_norm(Tensor residual, Tensor branch, Tensor? gate, Tensor scale, "
            "Tensor weight_branch, Tensor weight_output, float epsilon=9.9999999999999995e-07) -> (Tensor, Tensor)",
    }
    for name, schema in schemas.items():
        assert str(getattr(torch.ops.mops, name).default._schema) == schema


def test_operators_refuse_wrong_arguments():
    W, i, o = torch.zeros(5, 4), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="embedding_lookup is not implemented for device cpu"):
        mt.embedding_lookup(W, i)
    with pytest.raises(TypeError, match="All index tensors must be of type int32"):
        mt.embedding_lookup(W, i.long())
    with pytest.raises(TypeError, match="only float32, float64, float16 and bfloat16 are supported"):
        mt.embedding_lookup(W.to(torch.complex64), i)
    with pytest.raises(ValueError, match="Expected W to have 2 dimensions"):
        mt.embedding_lookup(W[0], i)
    with pytest.raises(ValueError, match="is not implemented for device cpu"):
        mt.grouped_matrix_product(W, torch.zeros(1, 4, 2), o)
    with pytest.raises(TypeError, match="All floating point tensors must be of the same dtype"):
        mt.grouped_matrix_product(W, torch.zeros(1, 4, 2, dtype=torch.float64), o)
    with pytest.raises(ValueError, match="Expected W to have 3 dimensions"):
        mt.grouped_matrix_product(W, W, o)
    with pytest.raises(TypeError, match="All index tensors must be of type int32"):
        mt.grouped_matrix_product(W, torch.zeros(1, 4, 2), o.long())
    v = torch.zeros(4)
    with pytest.raises(ValueError, match="gated_residual_norm is not implemented for device cpu"):
        mt.gated_residual_norm(W, W, None, v, v, v)
    with pytest.raises(ValueError, match="Expected gate to have 2 dimensions"):
        mt.gated_residual_norm(W, W, v, v, v, v)
    with pytest.raises(TypeError, match="All floating point tensors must be of the same dtype"):
        mt.gated_residual_norm(W, W.half(), None, v, v, v)


def test_front_end_refuses_wrong_arguments():
    W, i = np.zeros((5, 4)), np.zeros(3, np.int32)
    with pytest.raises(TypeError, match="Wrong dtype for indices in embedding_lookup"):
        mops_b200.embedding_lookup(W, np.zeros(3))
    with pytest.raises(ValueError, match="`W` must be a 2D array in embedding_lookup, got a 1D array instead"):
        mops_b200.embedding_lookup(W[0], i)
    with pytest.raises(TypeError, match="`scale` must be a number in embedding_lookup"):
        mops_b200.embedding_lookup(W, i, "2")
    with pytest.raises(TypeError, match="`n_rows` must be a scalar in embedding_lookup_vjp"):
        mops_b200.embedding_lookup_vjp(W, i, 2.5)
    with pytest.raises(ValueError, match="`W` must be a 3D array in grouped_matrix_product"):
        mops_b200.grouped_matrix_product(W, W, i)
    with pytest.raises(ValueError, match="`scale` must be a 1D array in gated_residual_norm"):
        mops_b200.gated_residual_norm(W, W, None, W, W[0], W[0])


def _array(shape, dtype="float32", stride=None, data=0x1000):
    """An array that is never read: shapes are checked before anything is launched."""
    from mops_b200 import _lib
    if stride is None:
        stride = [int(np.prod(shape[d + 1:])) for d in range(len(shape))]
    return _lib.make_array(data, dtype, shape, stride)


@pytest.mark.parametrize("name,arguments,message", [
    ("embedding_lookup", [_array((3, 4)), _array((5, 6)), _array((3,), "int32"), 1.0],
     "the sizes of W along dimension 1 and output along dimension 1 must match in cuda_embedding_lookup"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4)), _array((2,), "int32"), 1.0],
     "the sizes of indices along dimension 0 and output along dimension 0 must match"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4), "float64"), _array((3,), "int32"), 1.0],
     "Expected output to be of type float64 in cuda_embedding_lookup, found float32"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4), "int32"), _array((3,), "int32"), 1.0], "Wrong dtype for W"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4), stride=(1, 5)), _array((3,), "int32"), 1.0],
     "W must have a last dimension of stride 1"),
    ("embedding_lookup", [_array((3, 4), stride=(8, 1)), _array((5, 4)), _array((3,), "int32"), 1.0],
     "output must be contiguous"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4)), _array((3,), "float32"), 1.0],
     "Expected indices to be of type int32"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4), data=0x1002), _array((3,), "int32"), 1.0],
     "W is not aligned to its values"),
    ("embedding_lookup", [_array((3, 4)), _array((5, 4), data=0), _array((3,), "int32"), 1.0], "W has no data"),
    ("embedding_lookup_vjp", [_array((5, 4)), _array((3, 4)), _array((3,), "int32"), 1.0, 5],
     "padding_index 5 is not a row of W"),
    ("grouped_matrix_product", [_array((7, 3)), _array((7, 4)), _array((2, 5, 3)), _array((3,), "int32")],
     "the sizes of W along dimension 1 and A along dimension 1 must match in cuda_grouped_matrix_product"),
    ("grouped_matrix_product", [_array((7, 3)), _array((7, 4)), _array((2, 4, 3)), _array((2,), "int32")],
     "along dimension 0 and offsets along dimension 0 must match"),
    ("grouped_matrix_product", [_array((7, 3)), _array((7, 4)), _array((2, 4, 3), stride=(24, 6, 2)), _array((3,), "int32")],
     "W must have a stride of 1 in one of its last two dimensions"),
    ("grouped_matrix_product_vjp", [_array((7, 4)), _array((2, 4, 2)), _array((7, 3)), _array((7, 4)), _array((2, 4, 3)),
                                    _array((3,), "int32")],
     "the sizes of W along dimension 2 and grad_W along dimension 2 must match"),
    ("gated_residual_norm", [_array((7, 4)), _array((7, 4)), _array((7, 4)), _array((7, 4)), _array((7, 2)), _array((4,)),
                             _array((4,)), _array((4,)), 1e-6],
     "gate must have as many columns as residual, or one"),
    ("gated_residual_norm", [_array((7, 4)), _array((7, 4)), _array((7, 4)), _array((6, 4)), _array((7, 1)), _array((4,)),
                             _array((4,)), _array((4,)), 1e-6],
     "the sizes of residual along dimension 0 and branch along dimension 0 must match"),
    ("gated_residual_norm", [_array((7, 4)), _array((7, 4)), _array((7, 4)), _array((7, 4)), _array((7, 1)), _array((4,)),
                             _array((4,)), _array((4,)), -1.0], "epsilon must not be negative"),
])
def test_entry_points_refuse_wrong_arrays(name, arguments, message):
    import ctypes
    from mops_b200 import _lib
    scalar = [ctypes.c_double(a) if isinstance(a, float) else ctypes.c_int64(a) if isinstance(a, int) else a
              for a in arguments]
    with pytest.raises(_lib.MopsError, match=message) as e:
        _lib.call(f"mops_b200_cuda_{name}", scalar)
    assert e.value.status == 1


# ======================================================================= embedding_lookup
def embedding_plain(W, indices, scale, grad, padding):
    W = W.double()
    n = torch.zeros(W.shape[0], device=W.device, dtype=torch.float64).index_add_(
        0, indices.long(), torch.ones(indices.numel(), device=W.device, dtype=torch.float64))
    keep = (indices != padding)[:, None]
    sums = torch.zeros_like(W).index_add_(0, indices.long(), grad.double() * keep)
    absolute = torch.zeros_like(W).index_add_(0, indices.long(), grad.double().abs() * keep)
    return W[indices.long()] * scale, sums * scale, absolute * abs(scale), n[:, None]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,rows,columns,padding", [
    (1, 1, 1, -1), (1, 70000, 8, -1), (2, 3, 1024, -1), (31, 5, 7, 2), (33, 4, 129, -1), (300, 300, 256, 0),
    (1000, 3, 40, 1), (4097, 257, 513, 256), (5000, 70001, 64, -1), (20000, 11, 96, 3), (9000, 1, 33, -1),
    (260, 9, 4096, -1), (16400, 2, 16, -1), (70000, 100, 24, 7)])
def test_embedding_matches_64_bits(dtype, tokens, rows, columns, padding):
    gen = torch.Generator(device="cuda").manual_seed(tokens * 7 + columns)
    W, grad = normal((rows, columns), dtype, 1).requires_grad_(True), normal((tokens, columns), dtype, 2)
    # many tokens at few rows
    u = torch.rand(tokens, generator=gen, device="cuda", dtype=torch.float64)
    indices = ((rows ** u).floor().clamp(0, rows - 1)).to(torch.int32)
    output = mt.embedding_lookup(W, indices, 1.75, padding)
    got, = torch.autograd.grad(output, [W], grad)
    want, sums, absolute, n = embedding_plain(W.detach(), indices, 1.75, grad, padding)
    close(output.detach(), want, want.abs(), 1, "output")
    close(got, sums, absolute, n, "grad_W")
    again, = torch.autograd.grad(mt.embedding_lookup(W, indices, 1.75, padding), [W], grad)
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("columns", [2, 6, 12, 20, 34, 258])
def test_embedding_rows_of_8_and_4_bytes(dtype, columns):
    W, grad = normal((61, columns), dtype, 1).requires_grad_(True), normal((700, columns), dtype, 2)
    indices = (torch.arange(700, device="cuda", dtype=torch.int32) * 7) % 53
    output = mt.embedding_lookup(W, indices, 1.75)
    got, = torch.autograd.grad(output, [W], grad)
    want, sums, absolute, n = embedding_plain(W.detach(), indices, 1.75, grad, -1)
    close(output.detach(), want, want.abs(), 1, "output")
    close(got, sums, absolute, n, "grad_W")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,rows,columns", [(3, 40, 1), (0, 33, 7), (50, 5000, 3), (20, 300, 1586), (700, 90000, 5), (17000, 70001, 3), (17001, 300, 33),
                                                 (16500, 90000, 8)])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_embedding_gradient_clears_every_row_wherever_it_begins(dtype, tokens, rows, columns, shift):
    import ctypes
    from mops_b200 import _lib
    gen = torch.Generator(device="cuda").manual_seed(rows + columns)
    indices = torch.randint(rows, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    grad = normal((tokens, columns), dtype, 2)
    room = torch.full((rows * columns + 16,), 7.0, dtype=dtype, device="cuda")
    got = room[shift:shift + rows * columns].view(rows, columns)
    array = lambda t: _lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), t.stride())
    torch.cuda.synchronize()
    _lib.call("mops_b200_cuda_embedding_lookup_vjp", [array(got), array(grad), array(indices), ctypes.c_double(1.0), ctypes.c_int64(-1)])
    sums = torch.zeros(rows, columns, dtype=torch.float64, device="cuda").index_add_(0, indices.long(), grad.double())
    absolute = torch.zeros_like(sums).index_add_(0, indices.long(), grad.double().abs())
    close(got, sums, absolute, max(int(torch.bincount(indices, minlength=1).max()), 1), "grad_W")
    assert (room[:shift] == 7).all() and (room[shift + rows * columns:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_embedding_on_strided_and_shifted_tensors(dtype):
    base = normal((50, 80), dtype, 3)
    indices = torch.arange(37, device="cuda", dtype=torch.int32) % 50
    for W in (base[:, 8:40], base[:, 3:40], base[:, ::2], base[::2, :33], base.T[:40]):
        part = indices % W.shape[0]
        assert torch.equal(mt.embedding_lookup(W, part, 2.0), W[part.long()] * 2)
    W = normal((50, 32), dtype, 4).requires_grad_(True)
    for grad in (base[:37, 8:40], base[:37, 3:35], base[:37, ::2][:, :32], base[:1, :32].expand(37, 32)):
        got, = torch.autograd.grad(mt.embedding_lookup(W, indices), [W], grad)
        want = torch.zeros(50, 32, device="cuda", dtype=torch.float64).index_add_(0, indices.long(), grad.double())
        close(got, want, want.abs(), 1)
    long = torch.arange(74, device="cuda", dtype=torch.int32)[::2] % 50
    assert torch.equal(mt.embedding_lookup(W, long).detach(), W.detach()[long.long()])


@pytest.mark.gpu
def test_embedding_empty_and_out_of_range():
    W = normal((6, 5), torch.float32, 5).requires_grad_(True)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    output = mt.embedding_lookup(W, none)
    assert output.shape == (0, 5)
    assert torch.equal(torch.autograd.grad(output, [W], output.detach())[0], torch.zeros_like(W))
    assert mt.embedding_lookup(W[:, :0], torch.zeros(3, dtype=torch.int32, device="cuda")).shape == (3, 0)
    bad = torch.tensor([1, -1, 5, 6, 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    output = mt.embedding_lookup(W, bad)  # not waited for: rows of zeros, no gradient
    want = torch.zeros(7, 5, device="cuda")
    want[[0, 2, 4]] = W.detach()[[1, 5, 1]]
    assert torch.equal(output.detach(), want)
    got, = torch.autograd.grad(output, [W], torch.ones_like(output))
    counts = torch.zeros(6, 5, device="cuda")
    counts[1], counts[5] = 2, 1
    assert torch.equal(got, counts)
    with pytest.raises(mops_b200.MopsError, match="Index array indices in operation cuda_embedding_lookup contains"):
        mops_b200.embedding_lookup(W.detach(), bad)
    with pytest.raises(mops_b200.MopsError, match="Index array indices in operation cuda_embedding_lookup_vjp"):
        mops_b200.embedding_lookup_vjp(output.detach(), bad, 6)
    # the next call is not affected, nor is one without rows
    assert torch.equal(mops_b200.embedding_lookup(W.detach(), bad[:1]), W.detach()[1:2])
    with pytest.raises(ValueError, match="padding_index 6 is not a row of W"):
        mt.embedding_lookup(W, none, 1.0, 6)


@pytest.mark.gpu
def test_embedding_keeps_infinities_where_they_are():
    W = torch.tensor([[1.0, float("inf")], [float("nan"), 2.0], [3.0, 4.0]], device="cuda")
    assert torch.equal(mt.embedding_lookup(W, torch.tensor([2, 0], dtype=torch.int32, device="cuda"), 2.0),
                       torch.tensor([[6.0, 8.0], [2.0, float("inf")]], device="cuda"))
    grad = torch.tensor([[float("inf"), 1.0], [2.0, float("nan")], [5.0, 6.0]], device="cuda")
    got = mops_b200.embedding_lookup_vjp(grad, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), 4, 1.0, 1)
    want = torch.tensor([[float("inf"), 1.0], [0.0, 0.0], [5.0, 6.0], [0.0, 0.0]], device="cuda")
    assert torch.equal(got, want)


# ================================================================= grouped_matrix_product
def grouped_plain(A, W, offsets, grad):
    A, W, grad = A.double(), W.double(), grad.double()
    outputs = [torch.zeros(A.shape[0], W.shape[2], device=A.device, dtype=torch.float64), torch.zeros_like(A), torch.zeros_like(W)]
    bounds = offsets.tolist()
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        outputs[0][lo:hi] = A[lo:hi] @ W[g]
        outputs[1][lo:hi] = grad[lo:hi] @ W[g].T
        outputs[2][g] = A[lo:hi].T @ grad[lo:hi]
    return outputs


def offsets_of(rows):
    return torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")


def check_grouped(A, W, offsets, grad):
    A, W = A.requires_grad_(True), W.requires_grad_(True)
    output = mt.grouped_matrix_product(A, W, offsets)
    got = [output.detach(), *torch.autograd.grad(output, [A, W], grad)]
    plain = A.detach(), W.detach(), offsets, grad
    want = grouped_plain(*plain)
    terms = grouped_plain(plain[0].abs(), plain[1].abs(), offsets, grad.abs())
    longest = max([b - a for a, b in zip(offsets.tolist(), offsets.tolist()[1:])] + [1])
    for g, w, t, n, what in zip(got, want, terms, (A.shape[1], W.shape[2], longest), ("output", "grad_A", "grad_W")):
        close(g, w, t, n, what)
    again = mt.grouped_matrix_product(A, W, offsets)
    assert torch.equal(again, output)
    for a, b in zip(torch.autograd.grad(again, [A, W], grad), got[1:]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K,N", [
    ([1], 1, 1), ([1], 64, 64), ([3, 0, 5], 7, 9), ([0, 0, 4, 0], 16, 24), ([64, 64], 64, 128), ([63, 65, 1], 72, 136),
    ([128, 129, 127], 128, 256), ([200, 0, 1, 300], 264, 40), ([1] * 40, 32, 48), ([17, 700], 96, 520), ([2000], 8, 16),
    ([5, 1, 250], 509, 131), ([33, 31], 1030, 30), ([0, 0], 16, 16), ([1000, 1], 130, 258), ([7] * 70, 16, 16),
    ([3000, 0, 129, 2500], 136, 1000), ([1111, 4000], 600, 770), ([300, 5000], 1000, 264)])
def test_grouped_matches_64_bits(dtype, rows, K, N):
    R = sum(rows)
    check_grouped(normal((R, K), dtype, 1), normal((len(rows), K, N), dtype, 2, K ** -0.5), offsets_of(rows),
                  normal((R, N), dtype, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K,N", [([3] * 30, 96, 520), ([200, 0, 1, 300], 1000, 40), ([1, 2, 3], 1024, 72), ([5000, 300], 64, 264)])
def test_grouped_gives_the_same_bits_every_time(dtype, rows, K, N):
    """Many calls in a row: what the parts of a block hand to each other is never read too early or written over too soon."""
    A, W = normal((sum(rows), K), dtype, 1), normal((len(rows), K, N), dtype, 2, K ** -0.5)
    offsets, grad = offsets_of(rows), normal((sum(rows), N), dtype, 3)
    A, W = A.requires_grad_(True), W.requires_grad_(True)

    def step():
        output = mt.grouped_matrix_product(A, W, offsets)
        return [output.detach(), *torch.autograd.grad(output, [A, W], grad)]

    first, differ = step(), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        for x, y in zip(step(), first):
            differ += (x != y).any()
    assert differ.item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("other_way", [False, True])
@pytest.mark.parametrize("before,rows,after,K,N", [
    (0, [1], 0, 4096, 8), (1, [0, 2, 0], 2, 1096, 2056), (0, [1] * 20 + [0] * 30 + [12], 0, 584, 136), (3, [17, 0, 1], 4, 264, 392),
    (0, [32], 0, 2048, 264), (0, [9, 70, 0, 20], 1, 2120, 2072), (5, [60, 0, 63], 0, 2048, 40), (0, [2, 5, 1, 0, 3], 0, 1536, 1024),
    (0, [0, 0, 0], 7, 128, 128), (0, [33], 0, 2056, 2304)])
def test_grouped_few_rows(dtype, other_way, before, rows, after, K, N):
    """Single tokens: the depth is cut into parts, the rows of no group are zero."""
    R = before + sum(rows) + after
    W = normal((len(rows), N, K), dtype, 2, K ** -0.5).transpose(1, 2) if other_way else normal((len(rows), K, N), dtype, 2, K ** -0.5)
    check_grouped(normal((R, K), dtype, 1), W, offsets_of(rows) + before, normal((R, N), dtype, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("before,rows,K,N", [
    (0, [1] * 13 + [0] * 7 + [5], 175, 269), (2, [0, 3, 0, 0, 1], 1, 1), (0, [1, 2, 0, 1], 3, 5), (0, [2] * 30, 1001, 7), (1, [0, 0, 1, 0, 31] + [0] * 20, 67, 2051),
    (0, [0, 40] + [0] * 20, 130, 3)])
def test_grouped_few_rows_of_odd_matrices(dtype, before, rows, K, N):
    """Matrices whose rows begin anywhere are read as they are, and most of the gradients of matrices are zero."""
    R = before + sum(rows)
    check_grouped(normal((R, K), dtype, 1), normal((len(rows), K, N), dtype, 2, K ** -0.5), offsets_of(rows) + before, normal((R, N), dtype, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(5, 3), (24, 40), (129, 67)])
@pytest.mark.parametrize("shift", [1, 3, 5])
def test_grouped_few_rows_outputs_begin_anywhere(dtype, K, N, shift):
    from mops_b200 import _lib
    rows = [1, 0, 3, 0, 0, 2]
    G, R = len(rows), sum(rows)
    A, W, offsets, grad = normal((R, K), dtype, 1), normal((G, K, N), dtype, 2, K ** -0.5), offsets_of(rows), normal((R, N), dtype, 3)
    room = torch.full((G * K * N + R * K + R * N + 64,), 7.0, dtype=dtype, device="cuda")
    views, at = [], shift
    for shape in ((R, N), (R, K), (G, K, N)):
        views.append(room[at:at + int(np.prod(shape))].view(shape))
        at += int(np.prod(shape))
    array = lambda t: _lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), t.stride())
    torch.cuda.synchronize()
    _lib.call("mops_b200_cuda_grouped_matrix_product", [array(t) for t in (views[0], A, W, offsets)])
    _lib.call("mops_b200_cuda_grouped_matrix_product_vjp", [array(t) for t in (views[1], views[2], grad, A, W, offsets)])
    want = grouped_plain(A, W, offsets, grad)
    terms = grouped_plain(A.abs(), W.abs(), offsets, grad.abs())
    for g, w, t, n, what in zip(views, want, terms, (K, N, 3), ("output", "grad_A", "grad_W")):
        close(g, w, t, n, what)
    assert (room[:shift] == 7).all() and (room[at:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(64, 128), (72, 40), (33, 65)])
def test_grouped_matrices_stored_the_other_way(dtype, K, N):
    rows = [100, 0, 37, 260]
    W = normal((4, N, K), dtype, 4, K ** -0.5).transpose(1, 2)
    check_grouped(normal((397, K), dtype, 5), W, offsets_of(rows), normal((397, N), dtype, 6))
    assert mt.grouped_matrix_product(normal((397, K), dtype, 5), W, offsets_of(rows)).is_contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grouped_on_strided_and_shifted_tensors(dtype):
    rows = [70, 3, 140]
    offsets = offsets_of(rows)
    A, W, grad = normal((213, 300), dtype, 7), normal((3, 160, 200), dtype, 8, 0.1), normal((213, 300), dtype, 9)
    for a, w, g in ((A[:, :128], W[:, :128, :96], grad[:, :96]), (A[:, 8:136], W[:, 8:136, 8:104], grad[:, 16:112]),
                    (A[:, 3:131], W[:, 1:129, 5:101], grad[:, 1:97]), (A[:, ::2][:, :64], W[:, :64:, ::2], grad[:, ::3]),
                    (A[:, :128], W[:, :128, :96], grad[:1, :96].expand(213, 96)),
                    (A[:, :128].T.contiguous().T, W[:, :128, :96], grad[:, :96])):
        check_grouped(a.detach(), w.detach(), offsets, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_rows_of_no_group_and_empty_sizes(dtype):
    offsets = torch.tensor([5, 9, 9, 140], dtype=torch.int32, device="cuda")
    A, W, grad = normal((150, 64), dtype, 1), normal((3, 64, 72), dtype, 2), normal((150, 72), dtype, 3)
    # what stands in rows of no group does not matter
    A[:5], A[140:], grad[:5], grad[140:] = float("nan"), float("inf"), float("nan"), float("-inf")
    A.requires_grad_(True), W.requires_grad_(True)
    output = mt.grouped_matrix_product(A, W, offsets)
    gA, gW = torch.autograd.grad(output, [A, W], grad)
    plain = grouped_plain(A.detach(), W.detach(), offsets, grad)
    terms = grouped_plain(A.detach().abs(), W.detach().abs(), offsets, grad.abs())
    for got, want, t, n in zip((output.detach(), gA, gW), plain, terms, (64, 72, 131)):
        close(got, want, t, n)
    assert (output[:5] == 0).all() and (output[140:] == 0).all() and (gW[1] == 0).all()
    for R, G, K, N in ((0, 2, 4, 4), (6, 0, 4, 4), (6, 2, 0, 4), (6, 2, 4, 0)):
        o = torch.zeros(G + 1, dtype=torch.int32, device="cuda")
        if G:
            o[1:] = R
        a, w = normal((R, K), dtype, 1).requires_grad_(True), normal((G, K, N), dtype, 2).requires_grad_(True)
        out = mt.grouped_matrix_product(a, w, o)
        assert out.shape == (R, N) and (out == 0).all()
        for x, like in zip(torch.autograd.grad(out, [a, w], torch.ones_like(out), allow_unused=True), (a, w)):
            assert x is None or (x.shape == like.shape and (x == 0).all())


@pytest.mark.gpu
def test_grouped_reports_wrong_offsets():
    A, W = normal((20, 16), torch.float32, 1), normal((3, 16, 8), torch.float32, 2)
    for bad in ([0, 5, 4, 20], [-1, 5, 9, 20], [0, 5, 9, 21], [0, 2 ** 31 - 1, 9, 20]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        with pytest.raises(mops_b200.MopsError, match="Index array offsets in operation cuda_grouped_matrix_product"):
            mops_b200.grouped_matrix_product(A, W, offsets)
        with pytest.raises(mops_b200.MopsError, match="Index array offsets in operation cuda_grouped_matrix_product_vjp"):
            mops_b200.grouped_matrix_product_vjp(normal((20, 8), torch.float32, 3), A, W, offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_infinities_stay_in_their_rows(dtype):
    A, W = normal((300, 64), dtype, 1), normal((2, 64, 64), dtype, 2)
    offsets = offsets_of([130, 170])
    clean = mops_b200.grouped_matrix_product(A, W, offsets)
    dirty = A.clone()
    dirty[129], dirty[131, 5] = float("nan"), float("inf")
    got = mops_b200.grouped_matrix_product(dirty, W, offsets)
    rest = torch.ones(300, dtype=torch.bool, device="cuda")
    rest[129] = rest[131] = False
    assert torch.equal(got[rest], clean[rest]) and got[129].isnan().all() and not got[131].isfinite().any()
    grad = normal((300, 64), dtype, 3)
    _, clean_W = mops_b200.grouped_matrix_product_vjp(grad, A, W, offsets)
    _, got_W = mops_b200.grouped_matrix_product_vjp(grad, dirty, W, offsets)
    assert got_W[0].isnan().all()
    assert torch.equal(got_W[1, :5], clean_W[1, :5]) and torch.equal(got_W[1, 6:], clean_W[1, 6:])
    assert not got_W[1, 5].isfinite().any()


# ==================================================================== gated_residual_norm
def norm_plain(arguments, epsilon, grads):
    leaves = [None if t is None else t.detach().double().requires_grad_(True) for t in arguments]
    x, b, g, s, w, p = leaves
    y = x + s * w * (1.0 if g is None else torch.sigmoid(g)) * b / (b.pow(2).mean(1, keepdim=True) + epsilon).sqrt()
    h = p * y / (y.pow(2).mean(1, keepdim=True) + epsilon).sqrt()
    gradients = torch.autograd.grad([y, h], [t for t in leaves if t is not None], [t.double() for t in grads])
    return [y.detach(), h.detach(), *gradients]


# Each value of the rows comes from a few products and from sums over the row; those are added up in parts (the values of one
# thread, then a tree), of which none has over sqrt(C) + 32 values for these widths, so their relative errors are at most
# (sqrt(C) + 32) u. A few of them multiply, and differences are taken of terms that are no larger than the
# largest operand or result: 32 times that, times the largest of those, bounds a value, and as many times that as values are added up
# a sum over rows or columns.
def check_norm(arguments, epsilon, grads):
    leaves = [t for t in arguments if t is not None]
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in arguments]
    outputs = mt.gated_residual_norm(*args, epsilon)
    got = [t.detach() for t in outputs] + list(torch.autograd.grad(outputs, leaves, grads))
    want = norm_plain(arguments, epsilon, grads)
    R, C = arguments[0].shape
    u = SUM[arguments[0].dtype]
    sizes = want[2].abs().max() if R else 0.0
    scale = max(float(t.abs().max()) for t in want[:2] + [g.double() for g in grads]) if R * C else 0.0
    for g, w, what in zip(got, want, ("stream", "normed", *["gradient %d" % i for i in range(6)])):
        assert g.shape == w.shape, what
        if not g.numel():
            continue
        size = max(float(w.abs().max()), scale, float(sizes))
        many = R if g.dim() == 1 else C if g.shape[1] == 1 else 1
        bound = ROUND[g.dtype] * w.abs() + 32 * (C ** 0.5 + 32) * many * u * size + SMALLEST[g.dtype]
        error = (g.double() - w).abs()
        assert not (error > bound).any() and not error.isnan().any(), f"{what}: {(error - bound).max().item():.3e} over"
    again = mt.gated_residual_norm(*args, epsilon)
    for a, b in zip(list(again) + list(torch.autograd.grad(again, leaves, grads)), got):
        assert torch.equal(a, b)


def norm_arguments(R, C, gate, dtype):
    x, b = normal((R, C), dtype, 1, 2.0), normal((R, C), dtype, 2)
    g = None if gate == 0 else normal((R, 1 if gate == 1 else C), dtype, 3, 2.0)
    s, w, p = (normal((C,), dtype, 4 + i) * 0.2 + 1 for i in range(3))
    return [x, b, g, s, w, p], [normal((R, C), dtype, 7), normal((R, C), dtype, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [0, 1, 2])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 64), (3, 2), (5, 7), (2, 129), (300, 16), (77, 100), (9, 1000), (4, 1024), (3, 2049),
                                 (700, 512), (2, 8192), (3, 20000), (1, 33333), (1200, 40)])
def test_norm_matches_64_bits(dtype, gate, R, C):
    check_norm(*(lambda a: (a[0], 1e-5, a[1]))(norm_arguments(R, C, gate, dtype)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_on_strided_and_shifted_tensors(dtype):
    wide = [normal((41, 300), dtype, i) for i in range(5)]
    s, w, p = (normal((300,), dtype, 6 + i) * 0.2 + 1 for i in range(3))
    for cut in (slice(0, 128), slice(8, 200), slice(3, 100), slice(0, 300, 2)):
        for gate in (wide[2][:, cut], wide[2][:, :1], wide[2][:1, :1].expand(41, 1)):
            check_norm([wide[0][:, cut], wide[1][:, cut], gate, s[cut], w[cut], p[cut]], 1e-5,
                       [wide[3][:, cut], wide[4][:, cut]])
    check_norm([wide[0], wide[1][:1].expand(41, 300), None, s, w, p], 1e-5, [wide[3], wide[4][:1].expand(41, 300)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_zero_rows_empty_sizes_and_large_gates(dtype):
    arguments, grads = norm_arguments(6, 48, 2, dtype)
    arguments[1][2] = 0          # a block that gives nothing
    arguments[2][3], arguments[2][4] = 3e4, -3e4
    check_norm(arguments, 1e-5, grads)
    arguments[0][2] = 0          # and a stream of zeros
    outputs = mt.gated_residual_norm(*arguments, 1e-5)
    assert (outputs[0][2] == 0).all() and (outputs[1][2] == 0).all()
    for R, C in ((0, 8), (3, 0)):
        a, g = norm_arguments(R, C, 1, dtype)
        a = [t.requires_grad_(True) for t in a]
        out = mt.gated_residual_norm(*a)
        assert out[0].shape == (R, C) and out[1].shape == (R, C)
        for x, like in zip(torch.autograd.grad(out, a, g, allow_unused=True), a):
            assert x is None or (x.shape == like.shape and (x == 0).all())


@pytest.mark.gpu
def test_norm_infinities_stay_in_their_rows():
    arguments, _ = norm_arguments(9, 256, 2, torch.float32)
    clean = mt.gated_residual_norm(*arguments)
    arguments[0][3, 5], arguments[1][6, 7] = float("inf"), float("nan")
    got = mt.gated_residual_norm(*arguments)
    rest = [0, 1, 2, 4, 5, 7, 8]
    for a, b in zip(got, clean):
        assert torch.equal(a[rest], b[rest])
    assert got[0][3, 5].isinf() and got[0][6].isnan().all()


# ============================================================ what they have in common
def small_problems(dtype=torch.float64):
    indices = torch.tensor([0, 2, 2, 1, 0], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda")
    a, _ = norm_arguments(3, 5, 2, dtype)
    return [
        (lambda W: mt.embedding_lookup(W, indices, 0.7), [normal((4, 3), dtype, 1)]),
        (lambda A, W: mt.grouped_matrix_product(A, W, offsets), [normal((5, 3), dtype, 1), normal((3, 3, 4), dtype, 2)]),
        (lambda *a: mt.gated_residual_norm(*a, 1e-3), a),
        (lambda x, b, g, s, w, p: mt.gated_residual_norm(x, b, g, s, w, p, 1e-3), a[:2] + [a[2][:, :1].clone()] + a[3:]),
        (lambda x, b, s, w, p: mt.gated_residual_norm(x, b, None, s, w, p, 1e-3), a[:2] + a[3:]),
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
def test_other_streams_and_graphs():
    """Tensors made on one stream and used on another, and a captured pass replayed on new values."""
    A, W = normal((500, 64), torch.bfloat16, 1), normal((4, 64, 96), torch.bfloat16, 2)
    offsets = offsets_of([100, 0, 150, 250])
    table, indices = normal((900, 64), torch.bfloat16, 3), (torch.arange(500, device="cuda", dtype=torch.int32) * 7) % 900
    a, g = norm_arguments(500, 96, 2, torch.bfloat16)

    def everything():
        rows = mops_b200.torch.embedding_lookup(table, indices, 0.5)
        product = mt.grouped_matrix_product(rows + A, W, offsets)
        return mt.gated_residual_norm(a[0], product, *a[2:])

    want = [t.clone() for t in everything()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything()
    A.add_(1.0)
    graph.replay()
    fresh = everything()
    assert all(torch.equal(x, y) for x, y in zip(captured, fresh))
    assert not torch.equal(fresh[0], want[0])


@pytest.mark.gpu
def test_front_end_on_tensors_and_host_arrays():
    W, A = normal((30, 24), torch.float32, 1), normal((40, 24), torch.float32, 2)
    indices, offsets = torch.arange(40, device="cuda", dtype=torch.int64) % 30, offsets_of([10, 30])
    M, grad = normal((2, 24, 16), torch.float32, 3), normal((40, 16), torch.float32, 4)
    a, g = norm_arguments(12, 24, 1, torch.float32)
    calls = [
        (mops_b200.embedding_lookup, [W, indices, 1.5]),
        (mops_b200.embedding_lookup_vjp, [A, indices, 30, 1.5, 3]),
        (mops_b200.grouped_matrix_product, [A, M, offsets]),
        (mops_b200.grouped_matrix_product_vjp, [grad, A, M, offsets]),
        (mops_b200.gated_residual_norm, a),
        (mops_b200.gated_residual_norm_vjp, g + a),
    ]
    for f, arguments in calls:
        want = f(*arguments)
        host = f(*[t.cpu().numpy() if isinstance(t, torch.Tensor) else t for t in arguments])
        with mops_b200.HostQueue():
            queued = f(*[t.cpu().numpy() if isinstance(t, torch.Tensor) else t for t in arguments])
        single = not isinstance(want, tuple)
        for w, h, q in zip(*([x] if single else x for x in (want, host, queued))):
            assert isinstance(h, np.ndarray) and np.array_equal(w.cpu().numpy(), h) and np.array_equal(h, q)
    half = mops_b200.embedding_lookup(W.half(), indices.int())
    assert half.dtype == torch.float16 and torch.equal(half, W.half()[indices])
    assert mops_b200.grouped_matrix_product_vjp(grad, A, M, offsets, compute_grad_A=False)[0] is None
    assert mops_b200.gated_residual_norm_vjp(*g, *a[:2], None, *a[3:])[2] is None
