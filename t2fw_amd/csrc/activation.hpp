// The sigmoid and what is made of it, for the operators around the recurrences.  16-bit results: hardware exponential and reciprocal,
// off by 2^-22 each and by |z| 2^-24 for the exponential's argument, of which a result in 16 bits keeps 2^-12 or 2^-9.  32-bit results: the library's.
#pragma once
#include "common.hpp"

namespace t2fw {

template <bool FAST> __device__ __forceinline__ float sigmoid_of(float z) {
    return FAST ? __builtin_amdgcn_rcpf(1.0f + __expf(-z)) : 1.0f / (1.0f + expf(-z));
}
// The product as a 32-bit number, before it is rounded to 16 bits: in one instruction with the conversion it would be rounded once, or not, by
// what stands around it, and a token by itself would differ from the same one in a sequence
__device__ __forceinline__ float as_float(float v) {
    asm("" : "+v"(v));
    return v;
}
// z sigmoid(z), and its derivative
template <bool FAST> __device__ __forceinline__ float silu_of(float z) { return as_float(z * sigmoid_of<FAST>(z)); }
__device__ __forceinline__ float silu_slope(float z, float s) { return s * fmaf(z, 1.0f - s, 1.0f); }

}  // namespace t2fw
