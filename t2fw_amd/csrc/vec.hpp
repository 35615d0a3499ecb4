// Vectors of elements as they lie in memory: loads and stores of up to 16 bytes at any element's address, and the element
// types' conversions to the type that sums are carried in.
#pragma once
#include "common.hpp"

namespace t2fw {

// N elements.  A row of an odd width starts at an odd element: a load of 16 bytes from a 2-byte aligned address is one instruction
// all the same (global memory takes unaligned accesses on this architecture), so that rows need no edge of single elements
// at their start.
template <typename IO, int N> struct Vec {
    IO e[N];
};
template <typename IO, int N> __device__ __forceinline__ Vec<IO, N> load_vec(const IO *p) {
    Vec<IO, N> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <typename IO, int N> __device__ __forceinline__ void store_vec(IO *p, const Vec<IO, N> &v) { __builtin_memcpy(p, &v, sizeof(v)); }

// Conversions by the hardware's instructions; to 16 bits with rounding to the nearest
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }
__device__ __forceinline__ float widen(__bf16 v) { return (float)v; }
template <typename IO, typename Acc> __device__ __forceinline__ IO narrow(Acc v) { return (IO)v; }

}  // namespace t2fw
