// The 2-norm over all gradients of a model, and the gradients scaled to a largest norm:
//   n = sqrt(sum of g^2),   g <- g min(1, max_norm / (n + 1e-6)).
// Two launches for up to CLIP_TABLE arrays, whose addresses and sizes travel as kernel arguments.  The arrays one after the other are cut into
// equal shares, one for each workgroup (in pieces of CLIP_PIECE elements of one array), which leaves one sum; in the second launch
// every workgroup adds up all sums in the same order, so that the norm does not depend on the order of events.  Squares and sums
// are carried in double: the conversions and additions hide behind memory, and no square overflows.
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

// The array that holds a piece: the last one whose first piece is not after it (arrays are not empty)
__device__ __forceinline__ int array_of(const ClipTable &t, uint32_t piece) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= piece) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Calls run(array, first element, elements) for what a workgroup's share of the pieces has of each array
template <typename Run> __device__ __forceinline__ void for_share(const ClipTable &t, uint32_t share, uint32_t shares, const Run &run) {
    uint32_t piece = (uint32_t)((uint64_t)t.pieces * share / shares);
    const uint32_t end = (uint32_t)((uint64_t)t.pieces * (share + 1) / shares);
    if (piece >= end) return;
    for (int a = array_of(t, piece); piece < end; ++a) {
        const uint32_t of_array = (t.n[a] + CLIP_PIECE - 1) / CLIP_PIECE, last = t.first[a] + of_array < end ? t.first[a] + of_array : end;
        const uint32_t from = (piece - t.first[a]) * CLIP_PIECE, to = (last - t.first[a]) * CLIP_PIECE;
        run(a, from, (to < t.n[a] ? to : t.n[a]) - from);
        piece = last;
    }
}

// Elements 0 .. n - 1 of an array, by the whole workgroup: vectors of VEC, AHEAD of them at a time, and single ones
template <typename IO, int VEC, int AHEAD, typename Each, typename Single>
__device__ __forceinline__ void over(const IO *p, uint32_t n, const Each &each, const Single &single) {
    constexpr uint32_t STEP = CLIP_THREADS * VEC;
    uint32_t i = 0;
    for (; i + STEP * AHEAD <= n; i += STEP * AHEAD) {
        Vec<IO, VEC> v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u] = load_vec<IO, VEC>(p + i + u * STEP + threadIdx.x * VEC);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) each(i + u * STEP + threadIdx.x * VEC, v[u]);
    }
    for (i += threadIdx.x * VEC; i + VEC <= n; i += STEP) each(i, load_vec<IO, VEC>(p + i));
    // the elements after the last whole vector, which is the one this thread stands at
    for (; i < n; ++i) single(i, p[i]);
}

template <typename IO> __device__ __forceinline__ double squares_of(const IO *p, uint32_t n) {
    constexpr int VEC = 16 / sizeof(IO);
    double s = 0;
    over<IO, VEC, 8>(
        p, n,
        [&](uint32_t, const Vec<IO, VEC> &v) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const double d = (double)widen(v.e[i]);
                s = fma(d, d, s);
            }
        },
        [&](uint32_t, IO e) {
            const double d = (double)widen(e);
            s = fma(d, d, s);
        });
    return s;
}

__global__ __launch_bounds__(CLIP_THREADS) void clip_squares_kernel(ClipTable t, double *partials) {
    double s = 0;
    for_share(t, blockIdx.x, gridDim.x, [&](int a, uint32_t from, uint32_t n) {
        switch (t.src_type[a]) {
            case T2FW_F32: s += squares_of(static_cast<const float *>(t.src[a]) + from, n); break;
            case T2FW_F16: s += squares_of(static_cast<const _Float16 *>(t.src[a]) + from, n); break;
            case T2FW_BF16: s += squares_of(static_cast<const __bf16 *>(t.src[a]) + from, n); break;
            default: s += squares_of(static_cast<const double *>(t.src[a]) + from, n); break;
        }
    });
    s = block_sum(s);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// A product in double, whatever the types: a norm above float32's largest has a factor that 32 bits do not hold, and 64-bit gradients keep
// theirs.  16-bit results go by way of 32 bits.
template <typename B> __device__ __forceinline__ B scaled(double v, double by) {
    return sizeof(B) == 2 ? narrow<B>((float)(v * by)) : narrow<B>(v * by);
}
template <typename A, typename B> __device__ __forceinline__ void scale_share(const A *src, B *dst, uint32_t n, double by) {
    constexpr int VEC = 16 / (sizeof(A) > sizeof(B) ? sizeof(A) : sizeof(B));
    over<A, VEC, 8>(
        src, n,
        [&](uint32_t i, const Vec<A, VEC> &v) {
            Vec<B, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.e[j] = scaled<B>(widen(v.e[j]), by);
            store_past(dst + i, o);
        },
        [&](uint32_t i, A e) { dst[i] = scaled<B>(widen(e), by); });
}
template <typename A> __device__ __forceinline__ void scale_from(const A *src, void *dst, int dst_type, uint32_t at, uint32_t n, double by) {
    switch (dst_type) {
        case T2FW_F32: scale_share(src + at, static_cast<float *>(dst) + at, n, by); break;
        case T2FW_F16: scale_share(src + at, static_cast<_Float16 *>(dst) + at, n, by); break;
        case T2FW_BF16: scale_share(src + at, static_cast<__bf16 *>(dst) + at, n, by); break;
        default: scale_share(src + at, static_cast<double *>(dst) + at, n, by); break;
    }
}

__global__ __launch_bounds__(CLIP_THREADS) void clip_scale_kernel(ClipTable t, const double *partials, int total, double max_norm, float *norm) {
    double s = 0;
    for (int i = threadIdx.x; i < total; i += CLIP_THREADS) s += partials[i];
    const double n = sqrt(block_sum(s));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double ratio = max_norm / (n + 1e-6), by = ratio > 1.0 ? 1.0 : ratio;           // a norm that is NaN makes NaN of everything
    // From the last array to the first, and with stores that leave the last-level cache alone: it still holds much of what the sums have just
    // read.  119 M bf16 gradients into float32: 204 us with ordinary stores, 157 so (713 MB at the rate of a copy: 143).
    for_share(t, gridDim.x - 1 - blockIdx.x, gridDim.x, [&](int a, uint32_t from, uint32_t m) {
        // not wanted; or in place and within the limit: nothing changes
        if (t.dst[a] == nullptr || (by == 1.0 && t.dst[a] == t.src[a])) return;
        switch (t.src_type[a]) {
            case T2FW_F32: scale_from(static_cast<const float *>(t.src[a]), t.dst[a], t.dst_type[a], from, m, by); break;
            case T2FW_F16: scale_from(static_cast<const _Float16 *>(t.src[a]), t.dst[a], t.dst_type[a], from, m, by); break;
            case T2FW_BF16: scale_from(static_cast<const __bf16 *>(t.src[a]), t.dst[a], t.dst_type[a], from, m, by); break;
            default: scale_from(static_cast<const double *>(t.src[a]), t.dst[a], t.dst_type[a], from, m, by); break;
        }
    });
}

}  // namespace

int clip_squares(const ClipTable &t, int groups, double *partials, hipStream_t stream) {
    hipLaunchKernelGGL(clip_squares_kernel, dim3(groups), dim3(CLIP_THREADS), 0, stream, t, partials);
    return check_hip(hipGetLastError(), "clip_squares_kernel launch");
}

int clip_scale(const ClipTable &t, int groups, const double *partials, int total, double max_norm, float *norm, hipStream_t stream) {
    hipLaunchKernelGGL(clip_scale_kernel, dim3(groups), dim3(CLIP_THREADS), 0, stream, t, partials, total, max_norm, norm);
    return check_hip(hipGetLastError(), "clip_scale_kernel launch");
}

}  // namespace t2fw
