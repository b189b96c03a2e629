// The functions of gates, with their slopes, in 32 bits (f64: 64).
#ifndef MOPS_B200_ACTIVATION_CUH
#define MOPS_B200_ACTIVATION_CUH

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

} // namespace mops_b200

#endif
