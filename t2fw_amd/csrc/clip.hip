// The 2-norm over all gradients of a model, and the gradients scaled to a largest norm:
//   n = sqrt(sum of g^2),   g <- g min(1, max_norm / (n + 1e-6)).
// Two launches for up to CLIP_TABLE arrays, whose addresses and sizes travel as kernel arguments.  A workgroup takes chunks of
// CLIP_CHUNK elements in turn, whichever array they lie in, and leaves one sum; in the second launch every workgroup
// adds up all sums in the same order, so that the norm does not depend on the order of events.  Squares and sums are
// carried in double: the conversions and additions hide behind memory, and no square overflows.
#include "clip.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int CLIP_THREADS = 256;

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double parts[CLIP_THREADS / 64];
    v = group_sum(v, 64);
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < CLIP_THREADS / 64; ++i) v += parts[i];
    __syncthreads();
    return v;
}

// The array that holds a chunk: the last one whose first chunk is not after it (arrays are not empty)
__device__ __forceinline__ int array_of(const ClipTable &t, uint32_t chunk) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename IO> __device__ __forceinline__ double squares_of(const IO *p, uint32_t n) {
    constexpr int VEC = 16 / sizeof(IO), U = CLIP_CHUNK / (CLIP_THREADS * VEC);
    double s = 0;
    if (n == CLIP_CHUNK) {
        Vec<IO, VEC> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_vec<IO, VEC>(p + (u * CLIP_THREADS + threadIdx.x) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const double d = (double)widen(v[u].e[i]);
                s += d * d;
            }
        return s;
    }
    for (uint32_t i = threadIdx.x; i < n; i += CLIP_THREADS) {
        const double d = (double)widen(p[i]);
        s += d * d;
    }
    return s;
}

__global__ __launch_bounds__(CLIP_THREADS) void clip_squares_kernel(ClipTable t, double *partials) {
    double s = 0;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int a = array_of(t, c);
        const uint32_t at = (c - t.first[a]) * CLIP_CHUNK, left = t.n[a] - at, n = left < CLIP_CHUNK ? left : CLIP_CHUNK;
        switch (t.src_type[a]) {
            case T2FW_F32: s += squares_of(static_cast<const float *>(t.src[a]) + at, n); break;
            case T2FW_F16: s += squares_of(static_cast<const _Float16 *>(t.src[a]) + at, n); break;
            case T2FW_BF16: s += squares_of(static_cast<const __bf16 *>(t.src[a]) + at, n); break;
            default: s += squares_of(static_cast<const double *>(t.src[a]) + at, n); break;
        }
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

template <typename A, typename B> __device__ __forceinline__ void scale_chunk(const A *src, B *dst, uint32_t n, float by) {
    constexpr int VEC = 16 / (sizeof(A) > sizeof(B) ? sizeof(A) : sizeof(B)), U = CLIP_CHUNK / (CLIP_THREADS * VEC);
    if (n == CLIP_CHUNK) {
        Vec<A, VEC> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_vec<A, VEC>(src + (u * CLIP_THREADS + threadIdx.x) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Vec<B, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.e[i] = narrow<B>(widen(v[u].e[i]) * by);
            store_vec(dst + (u * CLIP_THREADS + threadIdx.x) * VEC, o);
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < n; i += CLIP_THREADS) dst[i] = narrow<B>(widen(src[i]) * by);
}
template <typename A> __device__ __forceinline__ void scale_from(const A *src, void *dst, int dst_type, uint32_t at, uint32_t n, float by) {
    switch (dst_type) {
        case T2FW_F32: scale_chunk(src + at, static_cast<float *>(dst) + at, n, by); break;
        case T2FW_F16: scale_chunk(src + at, static_cast<_Float16 *>(dst) + at, n, by); break;
        case T2FW_BF16: scale_chunk(src + at, static_cast<__bf16 *>(dst) + at, n, by); break;
        default: scale_chunk(src + at, static_cast<double *>(dst) + at, n, by); break;
    }
}

__global__ __launch_bounds__(CLIP_THREADS) void clip_scale_kernel(ClipTable t, const double *partials, int total, float max_norm, float *norm) {
    double s = 0;
    for (int i = threadIdx.x; i < total; i += CLIP_THREADS) s += partials[i];
    const float n = (float)sqrt(block_sum(s));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
    const float ratio = max_norm / (n + 1e-6f), by = ratio > 1.0f ? 1.0f : ratio;         // a norm that is NaN makes NaN of everything
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int a = array_of(t, c);
        // not wanted; or in place and within the limit: nothing changes
        if (t.dst[a] == nullptr || (by == 1.0f && t.dst[a] == t.src[a])) continue;
        const uint32_t at = (c - t.first[a]) * CLIP_CHUNK, left = t.n[a] - at, m = left < CLIP_CHUNK ? left : CLIP_CHUNK;
        switch (t.src_type[a]) {
            case T2FW_F32: scale_from(static_cast<const float *>(t.src[a]), t.dst[a], t.dst_type[a], at, m, by); break;
            case T2FW_F16: scale_from(static_cast<const _Float16 *>(t.src[a]), t.dst[a], t.dst_type[a], at, m, by); break;
            case T2FW_BF16: scale_from(static_cast<const __bf16 *>(t.src[a]), t.dst[a], t.dst_type[a], at, m, by); break;
            default: scale_from(static_cast<const double *>(t.src[a]), t.dst[a], t.dst_type[a], at, m, by); break;
        }
    }
}

}  // namespace

int clip_squares(const ClipTable &t, int groups, double *partials, hipStream_t stream) {
    hipLaunchKernelGGL(clip_squares_kernel, dim3(groups), dim3(CLIP_THREADS), 0, stream, t, partials);
    return check_hip(hipGetLastError(), "clip_squares_kernel launch");
}

int clip_scale(const ClipTable &t, int groups, const double *partials, int total, float max_norm, float *norm, hipStream_t stream) {
    hipLaunchKernelGGL(clip_scale_kernel, dim3(groups), dim3(CLIP_THREADS), 0, stream, t, partials, total, max_norm, norm);
    return check_hip(hipGetLastError(), "clip_scale_kernel launch");
}

}  // namespace t2fw
