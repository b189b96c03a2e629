"""grouped_matrix_product: operands that are infinite or NaN, whatever kernel multiplies them, the precision of deep f32 sums, and matrices of one row."""
import pytest
import torch

import mops_b200
import mops_b200.torch as mt
from mops_b200 import _lib
from test_block_ops import DTYPES, check_grouped, normal, offsets_of


def kinds(t):
    """0 for a number, else which of the other values."""
    return t.isnan().int() + 2 * (t == float("inf")).int() + 3 * (t == float("-inf")).int()


def check_infinities(rows, K, N, dtype, other_way):
    """Infinite and NaN operands at places of which some cancel, some meet a zero, and some lie beyond the first few hundred terms of a sum.
    What is not a number has to be what the sum of the products is; everything else keeps its bits."""
    R, G = sum(rows), len(rows)
    inf, nan = float("inf"), float("nan")
    A, grad = normal((R, K), dtype, 1), normal((R, N), dtype, 3)
    W = normal((G, N, K), dtype, 2, 0.2).transpose(1, 2) if other_way else normal((G, K, N), dtype, 2, 0.2)
    offsets = offsets_of(rows)
    run = lambda a, w, g: [mops_b200.grouped_matrix_product(a, w, offsets), *mops_b200.grouped_matrix_product_vjp(g, a, w, offsets)]
    clean = run(A, W, grad)
    A, W, grad = A.clone(), W.clone(), grad.clone()
    for t, at in ((A, [(0, 0, inf), (R - 1, K - 1, -inf), (R // 2, K // 2, inf), (R // 2, K // 3, -inf), (R // 3, 0, nan)]),
                  (grad, [(R - 1, 0, inf), (R // 3, N // 2, -inf), (0, N - 1, nan)])):
        for r, c, v in at:
            t[r, c] = v
    W[0, K - 1, 0], W[G - 1, 0, N - 1], W[0, K // 2, N // 3] = inf, -inf, 0.0
    got = run(A, W, grad)
    bounds = offsets.tolist()
    a, w, g = A.double(), W.double(), grad.double()
    want = [torch.zeros(R, N, dtype=torch.float64, device="cuda"), torch.zeros_like(a), torch.zeros_like(w)]
    # elementwise products and sums: a library's product may leave out what is multiplied by zero
    for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        for r in range(lo, hi):
            want[0][r] = (a[r, :, None] * w[i]).sum(0)
            want[1][r] = (w[i] * g[r]).sum(1)
        for k in range(K):
            want[2][i, k] = (a[lo:hi, k, None] * g[lo:hi]).sum(0)
    for x, y, before, what in zip(got, want, clean, ("output", "grad_A", "grad_W")):
        assert torch.equal(kinds(x.double()), kinds(y)), what
        same = (kinds(y) == 0)
        assert same.any() and not same.all(), what
    # rows and columns that hold none of them keep their bits
    keep = torch.ones(R, dtype=torch.bool, device="cuda")
    keep[[0, R // 3, R // 2, R - 1]] = False
    columns = torch.ones(N, dtype=torch.bool, device="cuda")
    columns[[0, N // 3, N - 1]] = False
    assert torch.equal(got[0][keep][:, columns], clean[0][keep][:, columns])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("other_way", [False, True])
@pytest.mark.parametrize("rows,K,N", [([3, 2], 40, 24), ([8], 128, 64), ([20, 15], 96, 48), ([150, 0, 90], 64, 128), ([150, 70], 129, 67), ([40, 300], 520, 200), ([5, 600], 72, 33),
                                      ([700], 40, 24), ([90, 161], 300, 130)])
def test_infinities_come_out_as_they_are(dtype, other_way, rows, K, N):
    check_infinities(rows, K, N, dtype, other_way)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 200])
def test_a_row_gives_the_same_infinities_alone_and_among_many(rows):
    """The kernels for few rows and those for many."""
    A = normal((rows, 64), torch.float32, 1)
    A[:, 7] = torch.where(torch.arange(rows, device="cuda") % 3 == 0, float("inf"), float("-inf"))
    W, offsets = normal((1, 64, 96), torch.float32, 2), offsets_of([rows])
    got = mops_b200.grouped_matrix_product(A, W, offsets)
    assert torch.equal(got, A[:, 7:8] * W[0, 7:8])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_operands_without_a_number(value):
    """Everything is computed again here."""
    A, grad = torch.full((1500, 700), value, device="cuda"), torch.ones(1500, 300, device="cuda")
    W, offsets = torch.ones(2, 700, 300, device="cuda"), offsets_of([1000, 500])
    got = [mops_b200.grouped_matrix_product(A, W, offsets), mops_b200.grouped_matrix_product_vjp(grad, A, W, offsets)[1]]
    for x in got:
        assert x.isnan().all() if value != value else (x == value).all()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["output", "output, depth in memory", "gradient of the matrices"])
@pytest.mark.parametrize("depth", [512, 8192])
def test_deep_sums_of_one_sign_in_f32(what, depth):
    """Values between 1 and 2, so that what is cut off a sum does not cancel: the error of a result is at most

    * 3 * 2^-23 of it for what splitting leaves out (three products of parts, each at most 2^-7 2^-16 of the leading one),
    * 24 additions to an accumulator of 64 values, each of which cuts less than two units of the accumulator's last place off (2^-22 of it): 24 * 2^-22, and
    * depth / 64 roundings of sums that grow from nothing: depth / 64 * 2^-24, and one more for parts that are joined.

    The second term would be depth / 64 times as large if an accumulator took the whole depth."""
    gen = torch.Generator(device="cuda").manual_seed(depth)
    values = lambda *shape: 1 + torch.rand(shape, generator=gen, device="cuda")
    offsets = offsets_of([160])
    if what == "gradient of the matrices":
        offsets = offsets_of([depth])
        A, grad = values(depth, 136), values(depth, 72)
        _, got = mops_b200.grouped_matrix_product_vjp(grad, A, values(1, 136, 72), offsets, compute_grad_A=False)
        got, want = got[0], A.double().T @ grad.double()
    else:
        A, W = values(160, depth), values(1, depth, 72)
        if what != "output":  # (as the gradient of a product's first operand)
            got, _ = mops_b200.grouped_matrix_product_vjp(A, values(160, 72), W.transpose(1, 2).contiguous(), offsets, compute_grad_W=False)
        else:
            got = mops_b200.grouped_matrix_product(A, W, offsets)
        want = A.double() @ W[0].double()
    bound = 3 * 2.0 ** -23 + 24 * 2.0 ** -22 + (depth / 64 + 1) * 2.0 ** -24
    assert ((got.double() - want).abs() / want).max().item() <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[2, 1], [70, 0, 200]])
@pytest.mark.parametrize("N", [1, 3, 40, 129])
def test_matrices_of_one_row_whose_columns_lie_apart(dtype, rows, N):
    """Strides of a dimension of one value mean nothing: with one column of a wider array the other way round, the only stride of 1 is such a one."""
    G, R = len(rows), sum(rows)
    wide = normal((G, N, 5), dtype, 1)
    W = wide[:, :, 2:3].transpose(1, 2)
    check_grouped(normal((R, 1), dtype, 2), W.detach(), offsets_of(rows), normal((R, N), dtype, 3))
    check_grouped(normal((R, N), dtype, 2), wide[:, :, 1:2].detach(), offsets_of(rows), normal((R, 1), dtype, 3))
    # through the C ABI
    A, offsets, out = normal((R, 1), dtype, 2), offsets_of(rows), torch.empty(R, N, dtype=dtype, device="cuda")
    array = lambda t, stride=None: _lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), stride or t.stride())
    torch.cuda.synchronize()
    for stride in (1, 7, 5 * N):
        out.fill_(7)
        torch.cuda.synchronize()
        _lib.call("mops_b200_cuda_grouped_matrix_product", [array(out), array(A), array(W, (5 * N, stride, 5)), array(offsets)])
        assert torch.equal(out, mt.grouped_matrix_product(A, W.contiguous(), offsets))
