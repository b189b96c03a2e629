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
* ``grouped_gated_product(A, W, offsets, activation="silu")``: the gated feed-forward layer of each group, ``W`` of G x K x 2N with the gate's
  columns first: ``f(A[r] @ W[g][:, :N]) * (A[r] @ W[g][:, N:])``, f silu or gelu.
* ``linear_cross_entropy(A, W, targets, scale=1.0, ignore_index=-1)``: ``loss`` and ``log_sum`` of each row, of the logits
  ``scale * A @ W.T``, which are not kept. Rows whose target is ``ignore_index`` have zeros and no gradient.

And for all gradients of a model together, whose types may differ (not differentiable):

* ``gradient_norm(gradients)``: the root of the sum of squares of all their values.
* ``clip_gradient_norm(gradients, max_norm)``: that norm, and the gradients scaled to ``max_norm`` where it is larger;
  ``clip_gradient_norm_`` scales them in place and returns the norm. Where the norm is not finite they stay as they are.
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
grouped_gated_product = torch.ops.mops.grouped_gated_product
linear_cross_entropy = torch.ops.mops.linear_cross_entropy
gradient_norm = torch.ops.mops.gradient_norm
clip_gradient_norm = torch.ops.mops.clip_gradient_norm
clip_gradient_norm_ = torch.ops.mops.clip_gradient_norm_

__all__ = [
    "homogeneous_polynomial_evaluation",
    "sparse_accumulation_of_products",
    "outer_product_scatter_add",
    "outer_product_scatter_add_with_weights",
    "sparse_accumulation_scatter_add_with_weights",
    "embedding_lookup",
    "grouped_matrix_product",
    "gated_residual_norm",
    "grouped_gated_product",
    "linear_cross_entropy",
    "gradient_norm",
    "clip_gradient_norm",
    "clip_gradient_norm_",
]
