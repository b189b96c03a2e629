"""``torch.ops.mops.*`` backed by the sm_100a kernels.

Mirrors python/mops-torch/src/mops/torch/__init__.py of the reference: importing this module
loads the operator library, after which the five operations are available both as
``torch.ops.mops.<name>`` and as attributes of this module, differentiable through autograd
and usable from TorchScript. CUDA tensors only.

So are the operators of the block around them (no counterpart in the reference), for float32, float64,
float16 and bfloat16:

* ``embedding_lookup(W, indices, scale=1.0, padding_index=-1)``: ``scale * W[indices]``; the gradient of
  ``W`` leaves out ``padding_index``.
* ``grouped_matrix_product(A, W, offsets)``: ``A[r] @ W[g]`` for the rows ``offsets[g] <= r < offsets[g+1]``.
  ``W`` may be a transposed view (``weights.transpose(1, 2)``): nothing is copied.
* ``gated_residual_norm(residual, branch, gate, scale, weight_branch, weight_output, epsilon=1e-6)``:
  ``stream = residual + scale * weight_branch * sigmoid(gate) * branch / rms(branch)`` and
  ``weight_output * stream / rms(stream)``.
"""
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_HERE), "lib", "libmops_torch.so")

if not os.path.isfile(LIB_PATH):
    raise ImportError(f"{LIB_PATH} not found: build it with `python -m mops_b200.build`")
torch.ops.load_library(LIB_PATH)

homogeneous_polynomial_evaluation = torch.ops.mops.homogeneous_polynomial_evaluation
sparse_accumulation_of_products = torch.ops.mops.sparse_accumulation_of_products
outer_product_scatter_add = torch.ops.mops.outer_product_scatter_add
outer_product_scatter_add_with_weights = torch.ops.mops.outer_product_scatter_add_with_weights
sparse_accumulation_scatter_add_with_weights = (
    torch.ops.mops.sparse_accumulation_scatter_add_with_weights
)
embedding_lookup = torch.ops.mops.embedding_lookup
grouped_matrix_product = torch.ops.mops.grouped_matrix_product
gated_residual_norm = torch.ops.mops.gated_residual_norm

__all__ = [
    "homogeneous_polynomial_evaluation",
    "sparse_accumulation_of_products",
    "outer_product_scatter_add",
    "outer_product_scatter_add_with_weights",
    "sparse_accumulation_scatter_add_with_weights",
    "embedding_lookup",
    "grouped_matrix_product",
    "gated_residual_norm",
]
