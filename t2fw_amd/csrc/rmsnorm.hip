// The residual's addition and the root-mean-square norm of what is stored:
//   h = round(x + res) in the stream's type,  r = 1 / sqrt(mean h^2 + eps),  y = w h r;
//   backward, from dy and the stream's gradient dres:  u = w dy,  d_x = d_res = r (u - h r^2 mean(u h)) + dres,  d_w = sum over rows of dy h r.
// The norm is of the rounded h, the one that the backward finds again; sums are carried in 32 bits (64 for double).
// In 8 bits: y is divided by scale = max |y| / 448 of the row, or of each group of its columns, and rounded to float8 e4m3.
//
// A row stays in registers between its sums and its results: LANES threads hold it in chunks of 8 columns, CH of them each: 16 or 32
// lanes of a wave for narrow rows, a wave, or 4 to 16 waves.  Every load of a row is made before its sums, without a branch between
// them, also by lanes that have no columns left.  Where the width is no multiple of 8 the last chunk of a row is loaded
// from 8 columns before its end, and the columns that belong to the chunk before it are left out.
#include "rmsnorm.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int RN_THREADS = 256;
constexpr int RN_WIDTH = 8;              // columns of a chunk
constexpr float FP8_LARGEST = 448.0f;

template <typename IO> struct AccT { using type = float; };
template <> struct AccT<double> { using type = double; };

// Sums over the LANES threads of a row (part of a wave, one, or a workgroup of several)
template <int LANES, typename Acc> __device__ __forceinline__ void row_sums(Acc &v, Acc &u) {
    v = group_sum(v, LANES < 64 ? LANES : 64);
    u = group_sum(u, LANES < 64 ? LANES : 64);
    if (LANES > 64) {
        constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
        __shared__ Acc parts[2][WAVES];
        __syncthreads();
        if (threadIdx.x % 64 == 0) {
            parts[0][threadIdx.x / 64] = v;
            parts[1][threadIdx.x / 64] = u;
        }
        __syncthreads();
        v = u = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            v += parts[0][i];
            u += parts[1][i];
        }
    }
}
template <int LANES, typename Acc> __device__ __forceinline__ Acc row_sum(Acc v) {
    v = group_sum(v, LANES < 64 ? LANES : 64);
    if (LANES > 64) {
        constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
        __shared__ Acc parts[WAVES];
        __syncthreads();
        if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) v += parts[i];
    }
    return v;
}
// max that keeps a NaN
__device__ __forceinline__ float larger(float a, float b) { return a > b || a != a ? a : b; }
__device__ __forceinline__ float lanes_max(float v, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) v = larger(v, __shfl_xor(v, m, 64));
    return v;
}
template <int LANES> __device__ __forceinline__ float row_max(float v) {
    v = lanes_max(v, LANES < 64 ? LANES : 64);
    if (LANES > 64) {
        constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
        __shared__ float parts[WAVES];
        __syncthreads();
        if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) v = larger(v, parts[i]);
    }
    return v;
}

// 8 columns as they lie in memory
template <typename T> struct Eight {
    Raw16 raw[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) raw[i] = load_raw(p + i * (16 / sizeof(T)));
    }
    __device__ __forceinline__ float get(int i) const { return element<T>(raw[i / (16 / sizeof(T))], i % (16 / sizeof(T))); }
};
template <> struct Eight<double> {
    Vec<double, RN_WIDTH> v;
    __device__ __forceinline__ void load(const double *p) { v = load_vec<double, RN_WIDTH>(p); }
    __device__ __forceinline__ double get(int i) const { return v.e[i]; }
};

// A chunk of a row: its first column, where it is loaded from, how many of the loaded columns are not its own (8: it is past the end)
struct Chunk {
    int column, from, skip;
    __device__ __forceinline__ bool there() const { return skip < RN_WIDTH; }
};
__device__ __forceinline__ Chunk chunk_at(int index, int D) {
    Chunk c;
    c.column = index * RN_WIDTH;
    c.from = c.column + RN_WIDTH <= D ? c.column : D - RN_WIDTH;
    c.skip = c.column < D ? c.column - c.from : RN_WIDTH;
    return c;
}
template <typename T> __device__ __forceinline__ void store_chunk(T *row, const Chunk &c, const Vec<T, RN_WIDTH> &v) {
    if (c.skip == 0) {
        store_vec(row + c.from, v);
    } else if (c.there()) {
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i)
            if (i >= c.skip) row[c.from + i] = v.e[i];
    }
}
template <typename IO, typename Acc> __device__ __forceinline__ void load_weights(Acc (&o)[RN_WIDTH], const NormArgs &a, int from) {
    if (a.wide_w) {
        const Vec<float, RN_WIDTH> v = load_vec<float, RN_WIDTH>(static_cast<const float *>(a.w) + from);
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i) o[i] = v.e[i];
    } else {
        Eight<IO> v;
        v.load(static_cast<const IO *>(a.w) + from);
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i) o[i] = v.get(i);
    }
}

constexpr int threads_of(int lanes) { return lanes < RN_THREADS ? RN_THREADS : lanes; }

template <typename IO, typename Stream, int LANES, int CH, bool FP8>
__global__ __launch_bounds__(threads_of(LANES)) void norm_forward_kernel(NormArgs a) {
    using Acc = typename AccT<IO>::type;
    constexpr int ROWS = threads_of(LANES) / LANES;
    const int D = (int)a.D, lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES, base = (row < a.N ? row : a.N - 1) * a.D;
    const bool live = row < a.N;                         // (rows past the end compute with the last one, and store nothing)
    Chunk k[CH];
    Eight<IO> x[CH];
    Eight<Stream> res[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        k[c] = chunk_at(c * LANES + lane, D);
        x[c].load(static_cast<const IO *>(a.x) + base + k[c].from);
    }
    if (a.res != nullptr) {
#pragma unroll
        for (int c = 0; c < CH; ++c) res[c].load(static_cast<const Stream *>(a.res) + base + k[c].from);
    }
    Acc w[CH][RN_WIDTH], h[CH][RN_WIDTH], sum = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) load_weights<IO>(w[c], a, k[c].from);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Vec<Stream, RN_WIDTH> o;
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i) {
            h[c][i] = x[c].get(i);
            if (a.res != nullptr) h[c][i] += res[c].get(i);
            o.e[i] = narrow<Stream>(h[c][i]);
            h[c][i] = widen(o.e[i]);
            sum += i >= k[c].skip ? h[c][i] * h[c][i] : (Acc)0;
        }
        if (a.stored != nullptr && live) store_chunk(static_cast<Stream *>(a.stored) + base, k[c], o);
    }
    sum = row_sum<LANES>(sum);
    const Acc r = (Acc)1 / sqrt(sum / (Acc)a.D + (Acc)a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i) h[c][i] *= r * w[c][i];
    if constexpr (!FP8) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            Vec<IO, RN_WIDTH> o;
#pragma unroll
            for (int i = 0; i < RN_WIDTH; ++i) o.e[i] = narrow<IO>(h[c][i]);
            if (live) store_chunk(static_cast<IO *>(a.y) + base, k[c], o);
        }
    } else {
        float top[CH], all = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            top[c] = 0;
#pragma unroll
            for (int i = 0; i < RN_WIDTH; ++i)
                if (i >= k[c].skip) top[c] = larger(fabsf(h[c][i]), top[c]);
            all = larger(top[c], all);
        }
        const bool by_row = a.groups == 1;
        if (by_row) all = row_max<LANES>(all);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            // a group's chunks are neighbouring lanes of one wave, those past the end of the row among them
            float scale = (by_row ? all : lanes_max(top[c], (int)(a.group / RN_WIDTH))) / FP8_LARGEST;
            if (scale == 0.0f) scale = 1.0f;
            if (!live || !k[c].there()) continue;
            const int64_t g = by_row ? 0 : k[c].column / a.group;
            if (by_row ? lane == 0 && c == 0 : k[c].column % a.group == 0) a.scales[row * a.groups + g] = scale;
            // one reciprocal for the chunk; of a scale near the smallest numbers it would overflow
            const float by = 1.0f / scale;
            const bool tiny = scale < 1e-35f;
            uint32_t words[2];
#pragma unroll
            for (int i = 0; i < RN_WIDTH; i += 4) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = tiny ? h[c][i + j] / scale : h[c][i + j] * by;
                const int word = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
                words[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], word, true);
            }
            Vec<uint8_t, RN_WIDTH> o;
            __builtin_memcpy(&o, words, sizeof(o));
            store_chunk(static_cast<uint8_t *>(a.q) + base, k[c], o);
        }
    }
}

template <typename IO, typename Stream, int LANES, int CH>
__global__ __launch_bounds__(threads_of(LANES)) void norm_backward_kernel(NormArgs a) {
    using Acc = typename AccT<IO>::type;
    constexpr int THREADS = threads_of(LANES), ROWS = THREADS / LANES;
    const int D = (int)a.D, lane = threadIdx.x % LANES;
    Acc dw[CH][RN_WIDTH], w[CH][RN_WIDTH];
    Chunk k[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        k[c] = chunk_at(c * LANES + lane, D);
        load_weights<IO>(w[c], a, k[c].from);
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i) dw[c][i] = 0;
    }
    // (all rows of a workgroup go round together)
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < a.N; first += (int64_t)gridDim.x * ROWS) {
        const int64_t row = first + threadIdx.x / LANES, base = (row < a.N ? row : a.N - 1) * a.D;
        const bool live = row < a.N;
        Eight<Stream> h[CH], gr[CH];
        Eight<IO> u[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            h[c].load(static_cast<const Stream *>(a.stored) + base + k[c].from);
            u[c].load(static_cast<const IO *>(a.g_y) + base + k[c].from);
        }
        if (a.g_res != nullptr) {
#pragma unroll
            for (int c = 0; c < CH; ++c) gr[c].load(static_cast<const Stream *>(a.g_res) + base + k[c].from);
        }
        Acc squares = 0, dot = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < RN_WIDTH; ++i) {
                const Acc v = h[c].get(i);
                squares += i >= k[c].skip ? v * v : (Acc)0;
                dot += i >= k[c].skip ? v * u[c].get(i) * w[c][i] : (Acc)0;
            }
        row_sums<LANES>(squares, dot);
        const Acc r = (Acc)1 / sqrt(squares / (Acc)a.D + (Acc)a.eps), back = dot * r * r / (Acc)a.D;
        const Acc counts = live ? r : (Acc)0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            Vec<IO, RN_WIDTH> o;
            Vec<Stream, RN_WIDTH> os;
#pragma unroll
            for (int i = 0; i < RN_WIDTH; ++i) {
                const Acc v = h[c].get(i), t = u[c].get(i);
                if (live) dw[c][i] += t * v * counts;
                Acc g = r * (t * w[c][i] - v * back);
                if (a.g_res != nullptr) g += gr[c].get(i);
                o.e[i] = narrow<IO>(g);
                os.e[i] = narrow<Stream>(g);
            }
            if (!live) continue;
            store_chunk(static_cast<IO *>(a.d_x) + base, k[c], o);
            if (a.d_res != nullptr) store_chunk(static_cast<Stream *>(a.d_res) + base, k[c], os);
        }
    }
    // a workgroup's share of d_w: that of its rows' lanes added up in order
    if constexpr (ROWS > 1) {
        __shared__ Acc sums[ROWS - 1][CH * RN_WIDTH][LANES];
        if (threadIdx.x >= LANES) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < RN_WIDTH; ++i) sums[threadIdx.x / LANES - 1][c * RN_WIDTH + i][lane] = dw[c][i];
        }
        __syncthreads();
        if (threadIdx.x >= LANES) return;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < RN_WIDTH; ++i)
#pragma unroll
                for (int r = 0; r < ROWS - 1; ++r) dw[c][i] += sums[r][c * RN_WIDTH + i][lane];
    }
    Acc *part = static_cast<Acc *>(a.partials) + (int64_t)blockIdx.x * a.D;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Vec<Acc, RN_WIDTH> o;
#pragma unroll
        for (int i = 0; i < RN_WIDTH; ++i) o.e[i] = dw[c][i];
        store_chunk(part, k[c], o);
    }
}

// Rows of any width, by one workgroup each: what is stored is read again from memory.  For very wide rows, and those of fewer than 8
// columns.
template <typename IO, typename Stream, bool FP8>
__global__ __launch_bounds__(RN_THREADS) void norm_forward_any_kernel(NormArgs a) {
    using Acc = typename AccT<IO>::type;
    const int64_t row = blockIdx.x, base = row * a.D;
    const IO *x = static_cast<const IO *>(a.x) + base;
    const Stream *res = static_cast<const Stream *>(a.res);
    auto value = [&](int64_t i) {
        Acc h = widen(x[i]);
        if (res != nullptr) h += (Acc)widen(res[base + i]);
        return (Acc)widen(narrow<Stream>(h));
    };
    auto weight = [&](int64_t i) { return a.wide_w ? (Acc)static_cast<const float *>(a.w)[i] : (Acc)widen(static_cast<const IO *>(a.w)[i]); };
    Acc sum = 0;
    for (int64_t i = threadIdx.x; i < a.D; i += RN_THREADS) {
        const Acc h = value(i);
        sum += h * h;
    }
    sum = row_sum<RN_THREADS>(sum);
    const Acc r = (Acc)1 / sqrt(sum / (Acc)a.D + (Acc)a.eps);
    if (FP8) {
        const int64_t group = a.groups == 1 ? a.D : a.group;
        for (int64_t g = 0; g < a.groups; ++g) {
            const int64_t end = (g + 1) * group < a.D ? (g + 1) * group : a.D;
            float top = 0;
            for (int64_t i = g * group + threadIdx.x; i < end; i += RN_THREADS) top = larger(fabsf((float)(value(i) * r * weight(i))), top);
            float scale = row_max<RN_THREADS>(top) / FP8_LARGEST;
            if (scale == 0.0f) scale = 1.0f;
            if (threadIdx.x == 0) a.scales[row * a.groups + g] = scale;
            for (int64_t i = g * group + threadIdx.x; i < end; i += RN_THREADS)
                static_cast<uint8_t *>(a.q)[base + i] =
                    (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32((float)(value(i) * r * weight(i)) / scale, 0.0f, 0, false) & 0xff);
        }
    } else {
        for (int64_t i = threadIdx.x; i < a.D; i += RN_THREADS) static_cast<IO *>(a.y)[base + i] = narrow<IO>(value(i) * r * weight(i));
    }
    if (a.stored != nullptr)
        for (int64_t i = threadIdx.x; i < a.D; i += RN_THREADS) static_cast<Stream *>(a.stored)[base + i] = narrow<Stream>(value(i));
}

template <typename IO, typename Stream> __global__ __launch_bounds__(RN_THREADS) void norm_backward_any_kernel(NormArgs a) {
    using Acc = typename AccT<IO>::type;
    Acc *part = static_cast<Acc *>(a.partials) + (int64_t)blockIdx.x * a.D;
    auto weight = [&](int64_t i) { return a.wide_w ? (Acc)static_cast<const float *>(a.w)[i] : (Acc)widen(static_cast<const IO *>(a.w)[i]); };
    for (int64_t i = threadIdx.x; i < a.D; i += RN_THREADS) part[i] = 0;
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
        const Stream *h = static_cast<const Stream *>(a.stored) + row * a.D, *gr = static_cast<const Stream *>(a.g_res);
        const IO *gy = static_cast<const IO *>(a.g_y) + row * a.D;
        Acc squares = 0, dot = 0;
        for (int64_t i = threadIdx.x; i < a.D; i += RN_THREADS) {
            const Acc v = widen(h[i]);
            squares += v * v;
            dot += v * (Acc)widen(gy[i]) * weight(i);
        }
        row_sums<RN_THREADS>(squares, dot);
        const Acc r = (Acc)1 / sqrt(squares / (Acc)a.D + (Acc)a.eps), back = dot * r * r / (Acc)a.D;
        for (int64_t i = threadIdx.x; i < a.D; i += RN_THREADS) {
            const Acc v = widen(h[i]), u = widen(gy[i]);
            Acc g = r * (u * weight(i) - v * back);
            if (gr != nullptr) g += (Acc)widen(gr[row * a.D + i]);
            part[i] += u * v * r;
            static_cast<IO *>(a.d_x)[row * a.D + i] = narrow<IO>(g);
            if (a.d_res != nullptr) static_cast<Stream *>(a.d_res)[row * a.D + i] = narrow<Stream>(g);
        }
    }
}

// d_w: the sum of all shares.  A workgroup takes 32 columns with 32 threads each, whose loads do not wait for one another.
constexpr int RW_THREADS = 1024, RW_COLUMNS = 32, RW_ROWS = RW_THREADS / RW_COLUMNS;
template <typename IO, typename Acc>
__global__ __launch_bounds__(RW_THREADS) void norm_weights_kernel(NormArgs a, int64_t shares) {
    __shared__ Acc sums[RW_ROWS][RW_COLUMNS];
    const int64_t column = (int64_t)blockIdx.x * RW_COLUMNS + threadIdx.x % RW_COLUMNS;
    const Acc *p = static_cast<const Acc *>(a.partials) + column;
    Acc s = 0;
    if (column < a.D) {
#pragma unroll 8
        for (int64_t i = threadIdx.x / RW_COLUMNS; i < shares; i += RW_ROWS) s += p[i * a.D];
    }
    sums[threadIdx.x / RW_COLUMNS][threadIdx.x % RW_COLUMNS] = s;
    __syncthreads();
    if (threadIdx.x >= RW_COLUMNS || column >= a.D) return;
#pragma unroll
    for (int i = 1; i < RW_ROWS; ++i) s += sums[i][threadIdx.x];
    if (a.wide_w) static_cast<float *>(a.d_w)[column] = (float)s;
    else static_cast<IO *>(a.d_w)[column] = narrow<IO>(s);
}

constexpr int64_t WIDEST = 16384;        // columns of a row in registers
bool in_registers(int64_t D) { return D >= RN_WIDTH && D <= WIDEST; }
// threads of a row (0: the kernels for any width), for chunks of one or two to a thread
int lanes_of(int64_t D) {
    return !in_registers(D) ? 0 : D <= 128 ? 16 : D <= 256 ? 32 : D <= 1024 ? 64 : D <= 2048 ? 256 : D <= 8192 ? 512 : 1024;
}
int64_t rows_of_group(int64_t D) { return lanes_of(D) == 0 ? 1 : threads_of(lanes_of(D)) / lanes_of(D); }
// Workgroups of the backward: one for each CU before any takes a second row, then as many as are on the chip at once, with four
// rows of each thread or more, as every workgroup leaves a row of 32-bit sums.
int64_t backward_groups(int64_t N, int64_t D) {
    const int64_t rows = rows_of_group(D), need = (N + rows - 1) / rows, few = need < 256 ? need : 256, many = need / 4;      // (CUs: 256)
    const int64_t most = 1024 * RN_THREADS / threads_of(lanes_of(D) ? lanes_of(D) : RN_THREADS);
    return many < few ? few : many < most ? many / 256 * 256 : most;
}
// A row's threads and chunks by its width
#define NORM_BY_WIDTH(RUN, ANY)                                                                                                     \
    do {                                                                                                                            \
        const int lanes = lanes_of(a.D);                                                                                            \
        const bool one = a.D <= (int64_t)lanes * RN_WIDTH;                                                                          \
        const dim3 threads(lanes == 0 ? RN_THREADS : threads_of(lanes));                                                            \
        if (lanes == 0) ANY;                                                                                                        \
        else if (lanes == 16) RUN(16, 1);                                                                                           \
        else if (lanes == 32) RUN(32, 1);                                                                                           \
        else if (lanes == 64 && one) RUN(64, 1);                                                                                    \
        else if (lanes == 64) RUN(64, 2);                                                                                           \
        else if (lanes == 256) RUN(256, 1);                                                                                         \
        else if (lanes == 512 && one) RUN(512, 1);                                                                                  \
        else if (lanes == 512) RUN(512, 2);                                                                                         \
        else RUN(1024, 2);                                                                                                          \
    } while (0)

template <typename IO, typename Stream, bool FP8> int forward_of(const NormArgs &a, hipStream_t stream) {
    const int64_t groups = (a.N + rows_of_group(a.D) - 1) / rows_of_group(a.D);
    if (groups > 0x7fffffff) return fail(T2FW_ERR_BAD_SHAPE, "norm: too many rows for one launch");
    const dim3 grid((unsigned)groups);
#define NORM_RUN(L, C) hipLaunchKernelGGL((norm_forward_kernel<IO, Stream, L, C, FP8>), grid, threads, 0, stream, a)
    NORM_BY_WIDTH(NORM_RUN, hipLaunchKernelGGL((norm_forward_any_kernel<IO, Stream, FP8>), grid, threads, 0, stream, a));
#undef NORM_RUN
    return check_hip(hipGetLastError(), "norm_forward_kernel launch");
}

template <typename IO, typename Stream> int backward_of(const NormArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    const int64_t groups = backward_groups(a.N, a.D);
    const dim3 grid((unsigned)groups);
    if (a.N > 0) {
#define NORM_RUN(L, C) hipLaunchKernelGGL((norm_backward_kernel<IO, Stream, L, C>), grid, threads, 0, stream, a)
        NORM_BY_WIDTH(NORM_RUN, hipLaunchKernelGGL((norm_backward_any_kernel<IO, Stream>), grid, threads, 0, stream, a));
#undef NORM_RUN
        const int rc = check_hip(hipGetLastError(), "norm_backward_kernel launch");
        if (rc) return rc;
    }
    hipLaunchKernelGGL((norm_weights_kernel<IO, Acc>), dim3((unsigned)((a.D + RW_COLUMNS - 1) / RW_COLUMNS)), dim3(RW_THREADS), 0, stream, a,
                       norm_partials(a.N, a.D));
    return check_hip(hipGetLastError(), "norm_weights_kernel launch");
}

template <typename IO> int forward_types(const NormArgs &a, hipStream_t stream) {
    if (a.q != nullptr) return a.wide_stream ? forward_of<IO, float, true>(a, stream) : forward_of<IO, IO, true>(a, stream);
    return a.wide_stream ? forward_of<IO, float, false>(a, stream) : forward_of<IO, IO, false>(a, stream);
}
template <typename IO> int backward_types(const NormArgs &a, hipStream_t stream) {
    return a.wide_stream ? backward_of<IO, float>(a, stream) : backward_of<IO, IO>(a, stream);
}

}  // namespace

int64_t norm_partials(int64_t N, int64_t D) { return backward_groups(N, D); }

int norm_forward(const NormArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return a.q != nullptr ? forward_of<float, float, true>(a, stream) : forward_of<float, float, false>(a, stream);
        case T2FW_F16: return forward_types<_Float16>(a, stream);
        case T2FW_BF16: return forward_types<__bf16>(a, stream);
    }
    return forward_of<double, double, false>(a, stream);
}

int norm_backward(const NormArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return backward_of<float, float>(a, stream);
        case T2FW_F16: return backward_types<_Float16>(a, stream);
        case T2FW_BF16: return backward_types<__bf16>(a, stream);
    }
    return backward_of<double, double>(a, stream);
}

}  // namespace t2fw
