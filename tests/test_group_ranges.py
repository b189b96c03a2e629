"""Offsets that descend or lie outside of the rows: the ranges that the kernels make of them, on the host, and the error that
the operators give."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mops_b200", "csrc")


def test_ranges_end_whatever_the_offsets_say(tmp_path):
    """All pairs of offsets around a few rows: every range is inside of them, and every row of no group is visited once."""
    source, program = tmp_path / "ranges.cpp", tmp_path / "ranges"
    source.write_text("""
        #include <cstdio>
        #include <vector>
        #include "group_ranges.hpp"
        using namespace mops_b200;
        int main() {
            const int64_t far[] = {INT32_MIN, INT32_MAX};
            for (int64_t rows = 0; rows < 10; rows++) {
                std::vector<int64_t> ends(far, far + 2);
                for (int64_t v = -3; v < rows + 4; v++) ends.push_back(v);
                for (int64_t first : ends)
                    for (int64_t last : ends) {
                        const RowRange r = rows_between(first, last, rows);
                        if (r.lo < 0 || r.lo > r.hi || r.hi > rows) return printf("range of %d, %d\\n", int(first), int(last)), 1;
                        std::vector<int> seen(rows, 0);
                        int64_t visits = 0;
                        for_rows_of_no_group(first, last, rows, [&](int64_t row) {
                            if (row < 0 || row >= rows || ++visits > rows) throw "a visit too many";
                            seen[row]++;
                        });
                        for (int64_t row = 0; row < rows; row++)
                            if (seen[row] != (row < first || row >= last || first >= rows || last <= first)) return printf("row %d of %d, %d\\n", int(row), int(first), int(last)), 1;
                    }
            }
            return 0;
        }
    """)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(source), "-o", str(program)], check=True)
    subprocess.run([str(program)], check=True, timeout=60)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float64", "float16", "bfloat16"])
@pytest.mark.parametrize("K,N", [(64, 136), (33, 65)])
@pytest.mark.parametrize("other_way", [False, True])
def test_few_rows_report_offsets_that_descend(dtype, K, N, other_way):
    """Single tokens, whose kernels clear the rows of no group: in front of the first offset and behind the last one."""
    import torch

    import mops_b200
    dtype = getattr(torch, dtype)
    A, grad = torch.ones(8, K, dtype=dtype, device="cuda"), torch.ones(8, N, dtype=dtype, device="cuda")
    W = torch.ones(3, N, K, dtype=dtype, device="cuda").transpose(1, 2) if other_way else torch.ones(3, K, N, dtype=dtype, device="cuda")
    for bad in ([5, 5, 5, 2], [5, 6, 7, 4], [8, 0, 0, 0], [2 ** 31 - 1, 0, 0, -2 ** 31], [3, 1, 8, 3], [7, 0, 8, -1]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        with pytest.raises(mops_b200.MopsError, match="Index array offsets in operation cuda_grouped_matrix_product "):
            mops_b200.grouped_matrix_product(A, W, offsets)
        with pytest.raises(mops_b200.MopsError, match="Index array offsets in operation cuda_grouped_matrix_product_vjp"):
            mops_b200.grouped_matrix_product_vjp(grad, A, W, offsets)
    good = torch.tensor([1, 1, 3, 8], dtype=torch.int32, device="cuda")
    want = torch.full((8, N), float(K), dtype=dtype, device="cuda")
    want[0] = 0
    assert torch.equal(mops_b200.grouped_matrix_product(A, W, good), want)
