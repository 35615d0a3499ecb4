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

// The same past the last-level cache, for results that are not read soon where what is in there still is
template <typename IO, int N> __device__ __forceinline__ void store_past(IO *p, const Vec<IO, N> &v) {
    static_assert(sizeof(v) % 4 == 0, "whole words");
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(v) / 4), aligned(sizeof(IO))));
    Words w;
    __builtin_memcpy(&w, &v, sizeof(v));
    __builtin_nontemporal_store(w, reinterpret_cast<Words *>(p));
}

// Conversions by the hardware's instructions; to 16 bits with rounding to the nearest
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }
__device__ __forceinline__ float widen(__bf16 v) { return (float)v; }
template <typename IO, typename Acc> __device__ __forceinline__ IO narrow(Acc v) { return (IO)v; }

// 16 bytes of elements as they came, for what is held long and used several times: as elements of their own, 16-bit ones would take a
// register each.
struct Raw16 {
    uint32_t w[4];
};
__device__ __forceinline__ Raw16 load_raw(const void *p) {
    Raw16 r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename IO> __device__ __forceinline__ float element_of(const uint32_t *w, int j);
template <> __device__ __forceinline__ float element_of<float>(const uint32_t *w, int j) { return __uint_as_float(w[j]); }
template <> __device__ __forceinline__ float element_of<__bf16>(const uint32_t *w, int j) {
    return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
}
template <> __device__ __forceinline__ float element_of<_Float16>(const uint32_t *w, int j) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(j % 2 ? w[j / 2] >> 16 : w[j / 2]));
}
template <typename IO> __device__ __forceinline__ float element(const Raw16 &r, int j) { return element_of<IO>(r.w, j); }

}  // namespace t2fw
