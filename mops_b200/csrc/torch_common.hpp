// What the files of the torch operator library share: checks of arguments, the library's view of a tensor, and calls
// on torch's current stream.
#ifndef MOPS_B200_TORCH_COMMON_HPP
#define MOPS_B200_TORCH_COMMON_HPP

#include <string>
#include <vector>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/script.h>

#include "../../include/mops.h"
#include "mops.hpp"

namespace mops_torch {

using torch::Tensor;
using torch::autograd::AutogradContext;
using tensor_list = std::vector<Tensor>;

inline void same_device(const tensor_list& tensors) {
    for (const auto& t : tensors) {
        if (t.device() != tensors[0].device()) {
            C10_THROW_ERROR(ValueError, "All tensors must be on the same device, found " +
                                            t.device().str() + " and " + tensors[0].device().str());
        }
    }
}

inline void floating(const tensor_list& tensors) {
    const auto dtype = tensors[0].dtype();
    if (dtype != torch::kF64 && dtype != torch::kF32) {
        C10_THROW_ERROR(TypeError, "Found dtype " + std::string(dtype.name()) +
                                       ", only float32 and float64 are supported");
    }
    for (const auto& t : tensors) {
        if (t.dtype() != dtype) {
            C10_THROW_ERROR(TypeError,
                            "All floating point tensors must be of the same dtype, found " +
                                std::string(t.dtype().name()) + " and " + std::string(dtype.name()));
        }
    }
}

inline void int32_indices(const tensor_list& tensors) {
    for (const auto& t : tensors) {
        if (t.dtype() != torch::kI32) {
            C10_THROW_ERROR(TypeError, "All index tensors must be of type int32, found " +
                                           std::string(t.dtype().name()));
        }
    }
}

inline void ndim(const Tensor& t, int64_t expected, const char* name, const char* op) {
    if (t.dim() != expected) {
        C10_THROW_ERROR(ValueError, std::string("Expected ") + name + " to have " +
                                        std::to_string(expected) + " dimensions, in " + op +
                                        ", found " + std::to_string(t.dim()));
    }
}

inline void cuda_only(const Tensor& t, const char* op) {
    if (!t.device().is_cuda()) {
        C10_THROW_ERROR(ValueError, std::string(op) + " is not implemented for device " +
                                        t.device().str() +
                                        ": this build of mops provides the CUDA (sm_100a) "
                                        "implementations only");
    }
}

template <typename T, size_t N> mops::Tensor<T, N> view(const Tensor& t) {
    mops::Tensor<T, N> out;
    out.data = t.defined() ? t.data_ptr<T>() : nullptr;
    for (size_t d = 0; d < N; d++) out.shape[d] = t.defined() ? static_cast<size_t>(t.size(d)) : 0;
    return out;
}

// Runs `body` with the device of `like` current and the library pointed at torch's current
// stream, without waiting for the kernels.
template <typename F> void on_stream_of(const Tensor& like, F&& body) {
    const c10::cuda::CUDAGuard guard(like.device());
    void* previous_stream = mops_b200_get_stream();
    const int previous_wait = mops_b200_get_wait();
    mops_b200_set_stream(at::cuda::getCurrentCUDAStream().stream());
    mops_b200_set_wait(0);
    try {
        body();
    } catch (...) {
        mops_b200_set_stream(previous_stream);
        mops_b200_set_wait(previous_wait);
        throw;
    }
    mops_b200_set_stream(previous_stream);
    mops_b200_set_wait(previous_wait);
}

inline Tensor maybe_empty_like(const Tensor& t) { return t.requires_grad() ? torch::empty_like(t) : Tensor(); }

// Outputs of an autograd Function must be defined tensors: a gradient that was not requested
// is returned as an empty placeholder and turned back into "no gradient" by the caller.
inline Tensor defined(const Tensor& t, const Tensor& like) {
    return t.defined() ? t : torch::empty({0}, like.options());
}
inline Tensor requested(const Tensor& t) { return t.defined() && t.numel() == 0 ? Tensor() : t; }

[[noreturn]] inline void no_second_derivative(const char* op) {
    C10_THROW_ERROR(NotImplementedError,
                    std::string("second derivatives are not supported in CUDA for ") + op);
}

// The gradients of an operation: through the differentiable Function when this backward pass is itself
// recorded (create_graph) or an argument carries a forward-mode tangent (which Function refuses, and
// which the kernels would drop), else straight from the kernels, without a node and saved variables
// that nobody would use.
template <typename Backward, typename... Args> tensor_list backward_of(const Args&... args) {
    const bool tangent = (... || (args.defined() && args._fw_grad(/*level=*/0).defined()));
    return at::GradMode::is_enabled() || tangent ? Backward::apply(args...) : Backward::run(args...);
}

} // namespace mops_torch

#endif
