// The functions of gates, with their slopes.
#ifndef MOPS_B200_ACTIVATION_CUH
#define MOPS_B200_ACTIVATION_CUH

#include <type_traits>

#include "../../include/mops.h"
#include "device.cuh"

namespace mops_b200 {

// silu: u sigmoid(u), slope s + u s (1 - s). gelu: u Phi(u), slope Phi(u) + u phi(u).
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

// Phi(u), given exp(-u^2 / 2), which its density is a multiple of. With z = |u| / sqrt(2) and t = 1 / (1 + 0.375 z), erfc(z) exp(z^2) is t times a polynomial of t of degree 8, fitted to the
// smallest relative error on 0 <= z <= 9.5 (1.1e-8; 1.5e-7 as it is evaluated), so that Phi keeps its figures where it is small. A third of the instructions of erfc and exp.
__device__ __forceinline__ float normal_distribution(float u, float density) {
    const float t = __fdividef(1.f, fmaf(0.375f * 0.70710678f, fabsf(u), 1.f));
    float q = 0.0616967715f;
    q = fmaf(q, t, -0.288076133f);
    q = fmaf(q, t, 0.43389535f);
    q = fmaf(q, t, -0.231078207f);
    q = fmaf(q, t, 0.274845332f);
    q = fmaf(q, t, 0.121038452f);
    q = fmaf(q, t, 0.205430552f);
    q = fmaf(q, t, 0.210633487f);
    q = fmaf(q, t, 0.211614415f);
    const float half = 0.5f * density * (t * q); // erfc(z) / 2
    return u < 0.f ? half : 1.f - half;
}

// f32.
template <int kActivation> struct Gate<kActivation, float> {
    float value, slope;
    __device__ __forceinline__ explicit Gate(float u) {
        if constexpr (kActivation == MOPS_B200_SILU) {
            const float s = __fdividef(1.f, 1.f + expf(-u)); // (0 where the exponential is beyond 2^126)
            value = u * s;
            slope = fmaf(value, 1.f - s, s);
        } else {
            // what the square is off by counts where it is large
            const float square = u * u, rest = fmaf(u, u, -square);
            const float density = expf(-0.5f * square) * (square < 1e30f ? fmaf(-0.5f, rest, 1.f) : 1.f), phi = normal_distribution(u, density);
            value = u * phi;
            slope = fmaf(u * 0.39894228f, density, phi);
        }
    }
};

// The same for results that are rounded to 16 bits: exponentials to some 2^-21.
template <int kActivation> struct FastGate {
    float value, slope;
    __device__ __forceinline__ explicit FastGate(float u) {
        if constexpr (kActivation == MOPS_B200_SILU) {
            const float s = __fdividef(1.f, 1.f + __expf(-u));
            value = u * s;
            slope = fmaf(value, 1.f - s, s);
        } else {
            const float density = __expf(-0.5f * u * u), phi = normal_distribution(u, density);
            value = u * phi;
            slope = fmaf(u * 0.39894228f, density, phi);
        }
    }
};

template <typename F> void for_activation(int32_t activation, F&& f) {
    if (activation == MOPS_B200_SILU) f(std::integral_constant<int, MOPS_B200_SILU>());
    else f(std::integral_constant<int, MOPS_B200_GELU>());
}

} // namespace mops_b200

#endif
