// Arrays of the block operators (embedding_lookup, grouped_matrix_product, gated_residual_norm): typed, strided views,
// as the C ABI passes them, and the checks that the operators make of them before anything is
// launched. The operators take f32, f64, f16 and bf16, which the reference's by-value structs cannot
// name, and rows that lie apart in memory (slices of a larger array), which saves a copy.
#ifndef MOPS_B200_ARRAYS_HPP
#define MOPS_B200_ARRAYS_HPP

#include <cstdint>
#include <stdexcept>
#include <string>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/mops.h"
#include "checks.hpp"
#include "device.cuh"

namespace mops_b200 {

using Array = mops_b200_array_t;

inline const char* type_name(int32_t type) {
    switch (type) {
    case MOPS_B200_F32: return "float32";
    case MOPS_B200_F64: return "float64";
    case MOPS_B200_F16: return "float16";
    case MOPS_B200_BF16: return "bfloat16";
    case MOPS_B200_I32: return "int32";
    default: return "an unknown type";
    }
}
inline int64_t type_bytes(int32_t type) {
    return type == MOPS_B200_F64 ? 8 : type == MOPS_B200_F16 || type == MOPS_B200_BF16 ? 2 : 4;
}

// Checks dimensions, sizes and that there is memory behind them; where a size is 1 or the array is empty, strides
// mean nothing and are replaced by those of a contiguous array.
inline void check_array(Array& a, const char* name, int dims, int32_t type, const std::string& op) {
    if (a.dimensions != dims)
        throw std::runtime_error(std::string("Expected ") + name + " to have " + std::to_string(dims) +
                                 " dimensions, in " + op + ", found " + std::to_string(a.dimensions));
    if (a.type != type)
        throw std::runtime_error(std::string("Expected ") + name + " to be of type " + type_name(type) + " in " + op +
                                 ", found " + type_name(a.type));
    int64_t values = 1;
    for (int d = 0; d < dims; d++) {
        if (a.shape[d] < 0)
            throw std::runtime_error("integer value '" + std::to_string(a.shape[d]) + "' does not fit in size_t");
        if (a.shape[d] > 0 && values > INT64_MAX / 16 / a.shape[d])
            throw std::runtime_error(std::string(name) + " is too large in " + op);
        values *= a.shape[d];
    }
    if (values > 0 && a.data == nullptr) throw std::runtime_error(std::string(name) + " has no data in " + op);
    if (reinterpret_cast<uintptr_t>(a.data) % type_bytes(type) != 0)
        throw std::runtime_error(std::string(name) + " is not aligned to its values in " + op);
    int64_t natural = 1;
    for (int d = dims - 1; d >= 0; d--) {
        if (values == 0 || a.shape[d] == 1) a.stride[d] = natural;
        if (a.stride[d] < 0) throw std::runtime_error(std::string(name) + " has a negative stride in " + op);
        natural *= a.shape[d] > 0 ? a.shape[d] : 1;
    }
}

inline void check_size(int64_t size, const char* name, int dim, int64_t expected, const char* other, int other_dim,
                       const std::string& op) {
    if (size != expected)
        throw std::runtime_error(std::string("Dimension mismatch: the sizes of ") + other + " along dimension " +
                                 std::to_string(other_dim) + " and " + name + " along dimension " +
                                 std::to_string(dim) + " must match in " + op);
}

// The last dimension of an input lies value by value in memory.
inline void check_rows(const Array& a, const char* name, const std::string& op) {
    const int last = a.dimensions - 1;
    if (a.shape[last] > 1 && a.stride[last] != 1)
        throw std::runtime_error(std::string(name) + " must have a last dimension of stride 1 in " + op);
}

// Outputs are contiguous: no two of their values may share a place.
inline void check_output(const Array& a, const char* name, const std::string& op) {
    int64_t natural = 1;
    for (int d = a.dimensions - 1; d >= 0; d--) {
        if (a.shape[d] > 1 && a.stride[d] != natural)
            throw std::runtime_error(std::string(name) + " must be contiguous in " + op);
        natural *= a.shape[d] > 0 ? a.shape[d] : 1;
    }
}

inline void check_floating(int32_t type, const char* name, const std::string& op) {
    if (type != MOPS_B200_F32 && type != MOPS_B200_F64 && type != MOPS_B200_F16 && type != MOPS_B200_BF16)
        throw std::runtime_error(std::string("Wrong dtype for ") + name + " in " + op + ": got " + type_name(type));
}

// Calls f with a value of the scalar type.
template <typename F> void for_type(int32_t type, F&& f) {
    switch (type) {
    case MOPS_B200_F32: f(float()); break;
    case MOPS_B200_F64: f(double()); break;
    case MOPS_B200_F16: f(__half()); break;
    default: f(__nv_bfloat16()); break;
    }
}

// Sums are held in 32 bits, of f64 in 64.
template <typename T> struct SumType { using type = float; };
template <> struct SumType<double> { using type = double; };
template <typename T> using Sum = typename SumType<T>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(Sum<T> v) { return static_cast<T>(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N values that are moved at once (16 bytes where N is 16 / sizeof(T), a single value where it is 1).
template <typename T, int N> struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
template <typename T> constexpr int kPack = 16 / static_cast<int>(sizeof(T));

// Writes what this call does not read again: the line goes to memory before others do.
template <typename T, int N> __device__ __forceinline__ void store_through(T* to, const Pack<T, N>& v) {
    if constexpr (N * sizeof(T) == 16) __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&v));
    else *reinterpret_cast<Pack<T, N>*>(to) = v;
}

// x / d for x < 2^32, by a multiplication: d times the rounded-up quotient 2^(32 + s) / d exceeds 2^(32 + s) by less than 2^s
// when 2^s >= d.
struct Divider {
    uint32_t d, shift;
    uint64_t factor;
    explicit Divider(uint32_t divisor) : d(divisor), shift(0) {
        while ((uint64_t(1) << shift) < d) shift++;
        factor = ((uint64_t(1) << (32 + shift)) + d - 1) / d;
    }
    __device__ __forceinline__ uint32_t divide(uint32_t x) const {
        return static_cast<uint32_t>((__umul64hi(factor << (31 - shift), uint64_t(x) << 1)));
    }
};

// Whether rows begin on multiples of so many bytes and are made of them.
inline bool aligned(const Array& a, int64_t to) {
    if (a.data == nullptr) return true;
    const int64_t bytes = type_bytes(a.type);
    bool ok = reinterpret_cast<uintptr_t>(a.data) % to == 0 && a.shape[a.dimensions - 1] * bytes % to == 0;
    for (int d = 0; d + 1 < a.dimensions; d++) ok = ok && a.stride[d] * bytes % to == 0;
    return ok;
}
inline bool aligned16(const Array& a) { return aligned(a, 16); }

template <typename T> inline const char* array_type_name() {
    return std::is_same<T, float>::value    ? "f32"
           : std::is_same<T, double>::value ? "f64"
           : std::is_same<T, __half>::value ? "f16"
                                            : "bf16";
}

} // namespace mops_b200

#endif
