// The block operators, as the C ABI calls them (the arguments are described in include/mops.h). Errors are thrown
// as std::runtime_error.
#ifndef MOPS_B200_BLOCK_OPS_HPP
#define MOPS_B200_BLOCK_OPS_HPP

#include "../../include/mops.h"

namespace mops_b200 {

using Array = mops_b200_array_t;

void embedding_lookup(Array output, Array W, Array indices, double scale);
void embedding_lookup_vjp(Array grad_W, Array grad_output, Array indices, double scale, int64_t padding_index);

void grouped_matrix_product(Array output, Array A, Array W, Array offsets);
void grouped_matrix_product_vjp(Array grad_A, Array grad_W, Array grad_output, Array A, Array W, Array offsets);

void gated_residual_norm(Array stream, Array normed, Array residual, Array branch, Array gate, Array scale,
                         Array weight_branch, Array weight_output, double epsilon);
void gated_residual_norm_vjp(Array grad_residual, Array grad_branch, Array grad_gate, Array grad_scale,
                             Array grad_weight_branch, Array grad_weight_output, Array grad_stream, Array grad_normed,
                             Array residual, Array branch, Array gate, Array scale, Array weight_branch,
                             Array weight_output, double epsilon);

void grouped_gated_product(Array output, Array A, Array W, Array offsets, int32_t activation);
void grouped_gated_product_vjp(Array grad_A, Array grad_W, Array grad_output, Array A, Array W, Array offsets, int32_t activation);

void linear_cross_entropy(Array loss, Array log_sum, Array A, Array W, Array targets, double scale, int64_t ignore_index);
void linear_cross_entropy_vjp(Array grad_A, Array grad_W, Array grad_loss, Array grad_log_sum, Array loss, Array log_sum, Array A, Array W,
                              Array targets, double scale, int64_t ignore_index);

void gradient_norm(Array norm, const Array* gradients, int64_t n);
void clip_gradient_norm(Array norm, const Array* outputs, const Array* gradients, int64_t n, double max_norm);

} // namespace mops_b200

#endif
