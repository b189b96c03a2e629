// The functions of gates, with their slopes, in 32 bits (f64: 64).
#ifndef MOPS_B200_ACTIVATION_CUH
#define MOPS_B200_ACTIVATION_CUH

#include <type_traits>

#include "../../include/mops.h"
#include "device.cuh"

namespace mops_b200 {

// silu: u sigmoid(u), slope s + u s (1 - s). gelu: u Phi(u), slope Phi(u) + u phi(u), Phi by erfc, which keeps its figures where Phi is small.
template <int kActivation, typename S> struct Gate {
    S value, slope;
    __device__ __forceinline__ explicit Gate(S u) {
        if constexpr (kActivation == MOPS_B200_SILU) {
            const S s = S(1) / (S(1) + exp(-u));
            value = u * s;
            slope = s + value * (S(1) - s);
        } else {
            const S phi = S(0.5) * erfc(u * S(-0.70710678118654752440));
            value = u * phi;
            slope = phi + u * (S(0.39894228040143267794) * exp(S(-0.5) * u * u));
        }
    }
};

// The same for results that are rounded to 16 bits: exponentials and quotients to some 2^-21.
template <int kActivation> struct FastGate {
    float value, slope;
    __device__ __forceinline__ explicit FastGate(float u) {
        if constexpr (kActivation == MOPS_B200_SILU) {
            const float s = __fdividef(1.f, 1.f + __expf(-u)); // (0 where the exponential is beyond 2^126)
            value = u * s;
            slope = fmaf(value, 1.f - s, s);
        } else {
            const Gate<kActivation, float> gate(u);
            value = gate.value, slope = gate.slope;
        }
    }
};

template <typename F> void for_activation(int32_t activation, F&& f) {
    if (activation == MOPS_B200_SILU) f(std::integral_constant<int, MOPS_B200_SILU>());
    else f(std::integral_constant<int, MOPS_B200_GELU>());
}

} // namespace mops_b200

#endif
