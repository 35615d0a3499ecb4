// The sigmoid and what is made of it, for the operators around the recurrences.  16-bit results: hardware exponential and reciprocal,
// off by 2^-22 each and by |z| 2^-24 for the exponential's argument, of which a result in 16 bits keeps 2^-12 or 2^-9.  32-bit results: the library's.
#pragma once
#include "common.hpp"

namespace t2fw {

template <bool FAST> __device__ __forceinline__ float sigmoid_of(float z) {
    return FAST ? __builtin_amdgcn_rcpf(1.0f + __expf(-z)) : 1.0f / (1.0f + expf(-z));
}
// z sigmoid(z), and its derivative
template <bool FAST> __device__ __forceinline__ float silu_of(float z) { return z * sigmoid_of<FAST>(z); }
__device__ __forceinline__ float silu_slope(float z, float s) { return s * fmaf(z, 1.0f - s, 1.0f); }

}  // namespace t2fw
