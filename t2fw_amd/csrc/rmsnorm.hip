// The residual's addition and the root-mean-square norm of what is stored:
//   h = round(x + res) in the stream's type,  r = 1 / sqrt(mean h^2 + eps),  y = w h r;
//   backward, from dy and the stream's gradient dres:  u = w dy,  d_x = d_res = r (u - h r^2 mean(u h)) + dres,  d_w = sum over rows of dy h r.
// The norm is of the rounded h, the one that the backward finds again; sums are carried in 32 bits (64 for double).
// In 8 bits: y is divided by scale = max |y| / 448 of the row, or of each group of its columns, and rounded to float8 e4m3.  r is in both and
// goes out: with p = (h 2^e) w, r = 2^e rest, 1 <= rest < 2, the code is that of 448 p / max |p|, rounded once, and
// scale = max |p| rest / 448.  A product of 16-bit numbers is exact in 32 bits.  What the rounding of others leaves out is carried for a stream of
// 32 bits, whose time it does not change (16384 x 8192: 325 us, without 322); next to a 16-bit stream, weights of 32 bits leave one
// code in a million at the other side of a middle (carried, 32768 x 4096 would take 233 us for 193).
//
// A row stays in registers between its sums and its results: LANES threads hold it in chunks of 16 bytes of the stream, CH of them each, so that a
// wave's loads and stores are of whole lines: 16 or 32 lanes of a wave for narrow rows, a wave, or 4 to 16 waves.  Every load of a row is made before its sums, without a branch between
// them, also by lanes that have no columns left.  Where the width is no multiple of a chunk the last one of a row is loaded
// from a chunk's width before its end, and the columns that belong to the chunk before it are left out.
//
// Bound by memory: 65536 x 1024 bf16 forward 111 us, backward 112 us with the weights' gradient (4.8 TB/s of four arrays each), 32768 x 4096
// in 8 bits 182 us (5.2 TB/s; a copy 5.0 to 5.4).  Rows of an odd width lose a fifth in 16-bit types, whose vectors are then
// not aligned (65536 x 1021: 130 and 126 us); aligned ones would start at another column in every row, and the backward's
// sums over the rows are per column.  64 x 768 in 8 bits: 4.9 us, one chain of loads, two sums over a wave and stores.
#include "rmsnorm.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int RN_THREADS = 256;
constexpr int RN_WIDTH = 8;              // columns of a thread, in one chunk or two
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
__device__ __forceinline__ float lanes_max(float v, int lanes) {          // of groups of 1 to 64 neighbouring lanes, as group_sum
    if (lanes >= 2) v = larger(v, dpp_move<DPP_QUAD_XOR1>(v));
    if (lanes >= 4) v = larger(v, dpp_move<DPP_QUAD_XOR2>(v));
    if (lanes >= 8) v = larger(v, dpp_move<DPP_ROW_HALF_MIRROR>(v));
    if (lanes >= 16) v = larger(v, dpp_move<DPP_ROW_MIRROR>(v));
    if (lanes >= 32) v = larger(v, __shfl_xor(v, 16, 64));
    if (lanes >= 64) v = larger(v, __shfl_xor(v, 32, 64));
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

// W columns as they lie in memory
template <typename T, int W> struct Piece {
    uint32_t w[sizeof(T) * W / 4];
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, p, sizeof(w)); }
    __device__ __forceinline__ float get(int i) const { return element_of<T>(w, i); }
};
template <int W> struct Piece<double, W> {
    Vec<double, W> v;
    __device__ __forceinline__ void load(const double *p) { v = load_vec<double, W>(p); }
    __device__ __forceinline__ double get(int i) const { return v.e[i]; }
};

// A chunk of a row: its first column, where it is loaded from, how many of the loaded columns are not its own (W: it is past the end)
template <int W> struct Chunk {
    int column, from, skip;
    __device__ __forceinline__ bool there() const { return skip < W; }
};
template <int W> __device__ __forceinline__ Chunk<W> chunk_at(int index, int D) {
    Chunk<W> c;
    c.column = index * W;
    c.from = c.column + W <= D ? c.column : D - W;
    c.skip = c.column < D ? c.column - c.from : W;
    return c;
}
template <typename T, int W> __device__ __forceinline__ void store_chunk(T *row, const Chunk<W> &c, const Vec<T, W> &v) {
    if (c.skip == 0) {
        store_vec(row + c.from, v);
    } else if (c.there()) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i >= c.skip) row[c.from + i] = v.e[i];
    }
}
template <typename IO, typename Acc, int W> __device__ __forceinline__ void load_weights(Acc (&o)[W], const NormArgs &a, int from) {
    if (a.wide_w) {
        const Vec<float, W> v = load_vec<float, W>(static_cast<const float *>(a.w) + from);
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = v.e[i];
    } else {
        Piece<IO, W> v;
        v.load(static_cast<const IO *>(a.w) + from);
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] = v.get(i);
    }
}

constexpr int threads_of(int lanes) { return lanes < RN_THREADS ? RN_THREADS : lanes; }

// r = power * rest with a power of two; a NaN stays in rest
__device__ __forceinline__ void parts_of(float r, float *power, float *rest) {
    const uint32_t bits = __float_as_uint(r);
    *power = __uint_as_float(bits & 0x7f800000u);
    *rest = r != r ? r : __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
}
__device__ __forceinline__ float scale_of(float top, float rest) {
    const float scale = top * rest / FP8_LARGEST;
    return scale == 0.0f ? 1.0f : scale;
}
// What the product of the largest lost in its rounding, of its absolute value; minus infinity from the others
__device__ __forceinline__ float lost_of(float h, float w, float top) {
    const float p = h * w, lost = fmaf(h, w, -p);
    return fabsf(p) == top ? p < 0 ? -lost : lost : -INFINITY;
}
// 448 h w / (top + lost), or 448 h / top, for W numbers: a product with the reciprocal, and from the remainder what it is off by.  For numbers whose
// reciprocal or remainder 32 bits do not hold, those that are not finite among them, y / scale.
template <int W, bool CARRIED>
__device__ __forceinline__ void codes_of(float (&v)[W], const float (&h)[W], const float (&w)[W], float top, float lost, float rest, float scale) {
    const float by = 1.0f / top, by448 = by * FP8_LARGEST;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float p = CARRIED ? h[i] * w[i] : h[i], q = p * by;
        float left = fmaf(-q, top, p);
        if (CARRIED) left = fmaf(-q, lost, left + fmaf(h[i], w[i], -p));
        v[i] = fmaf(q, FP8_LARGEST, left * by448);
    }
    if (__builtin_expect(!(scale >= 1e-33f && scale != 1.0f && top <= 1e35f), 0)) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = (CARRIED ? h[i] * w[i] : h[i]) * rest / scale;
    }
}

template <typename IO, typename Stream, int LANES, int CH, int W, bool FP8>
__global__ __launch_bounds__(threads_of(LANES)) void norm_forward_kernel(NormArgs a) {
    using Acc = typename AccT<IO>::type;
    constexpr int ROWS = threads_of(LANES) / LANES;
    const int D = (int)a.D, lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES, base = (row < a.N ? row : a.N - 1) * a.D;
    const bool live = row < a.N;                         // (rows past the end compute with the last one, and store nothing)
    Chunk<W> k[CH];
    Piece<IO, W> x[CH];
    Piece<Stream, W> res[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        k[c] = chunk_at<W>(c * LANES + lane, D);
        x[c].load(static_cast<const IO *>(a.x) + base + k[c].from);
    }
    if (a.res != nullptr) {
#pragma unroll
        for (int c = 0; c < CH; ++c) res[c].load(static_cast<const Stream *>(a.res) + base + k[c].from);
    }
    Acc w[CH][W], h[CH][W], sum = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) load_weights<IO, Acc, W>(w[c], a, k[c].from);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Vec<Stream, W> o;
#pragma unroll
        for (int i = 0; i < W; ++i) {
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
    if constexpr (!FP8) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            Vec<IO, W> o;
#pragma unroll
            for (int i = 0; i < W; ++i) o.e[i] = narrow<IO>(h[c][i] * (r * w[c][i]));
            if (live) store_chunk(static_cast<IO *>(a.y) + base, k[c], o);
        }
    } else {
        constexpr bool CARRIED = sizeof(Stream) > 2;     // else h becomes the product
        float top[CH], all = 0, power, rest;
        parts_of(r, &power, &rest);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            top[c] = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                h[c][i] *= power;
                if (!CARRIED) h[c][i] *= w[c][i];
                if (i >= k[c].skip) top[c] = larger(fabsf(CARRIED ? h[c][i] * w[c][i] : h[c][i]), top[c]);
            }
            all = larger(top[c], all);
        }
        const bool by_row = a.groups == 1;
        if (by_row) all = row_max<LANES>(all);
        float lost[CH], lost_all = -INFINITY;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            // (a group's chunks are neighbouring lanes of one wave, those past the end of the row among them)
            if (!by_row) top[c] = lanes_max(top[c], (int)(a.group / W));
            lost[c] = 0;
            if (!CARRIED) continue;
            lost[c] = -INFINITY;
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i >= k[c].skip) lost[c] = fmaxf(lost[c], lost_of(h[c][i], w[c][i], by_row ? all : top[c]));
            lost_all = fmaxf(lost_all, lost[c]);
            if (!by_row) lost[c] = lanes_max(lost[c], (int)(a.group / W));
        }
        if (CARRIED && by_row) lost_all = row_max<LANES>(lost_all);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const float largest = by_row ? all : top[c], scale = scale_of(largest, rest);
            if (!live || !k[c].there()) continue;
            const int64_t g = by_row ? 0 : k[c].column / a.group;
            if (by_row ? lane == 0 && c == 0 : k[c].column % a.group == 0) a.scales[row * a.groups + g] = scale;
            float v[W];
            codes_of<W, CARRIED>(v, h[c], w[c], largest, by_row ? lost_all : lost[c], rest, scale);
            uint32_t words[2];
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const int word = __builtin_amdgcn_cvt_pk_fp8_f32(v[i], v[i + 1], 0, false);
                words[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[i + 2], v[i + 3], word, true);
            }
            Vec<uint8_t, W> o;
            __builtin_memcpy(&o, words, sizeof(o));
            store_chunk(static_cast<uint8_t *>(a.q) + base, k[c], o);
        }
    }
}

template <typename IO, typename Stream, int LANES, int CH, int W>
__global__ __launch_bounds__(threads_of(LANES)) void norm_backward_kernel(NormArgs a) {
    using Acc = typename AccT<IO>::type;
    constexpr int THREADS = threads_of(LANES), ROWS = THREADS / LANES;
    const int D = (int)a.D, lane = threadIdx.x % LANES;
    Acc dw[CH][W], w[CH][W];
    Chunk<W> k[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        k[c] = chunk_at<W>(c * LANES + lane, D);
        load_weights<IO, Acc, W>(w[c], a, k[c].from);
#pragma unroll
        for (int i = 0; i < W; ++i) dw[c][i] = 0;
    }
    // (all rows of a workgroup go round together)
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < a.N; first += (int64_t)gridDim.x * ROWS) {
        const int64_t row = first + threadIdx.x / LANES, base = (row < a.N ? row : a.N - 1) * a.D;
        const bool live = row < a.N;
        Piece<Stream, W> h[CH], gr[CH];
        Piece<IO, W> u[CH];
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
            for (int i = 0; i < W; ++i) {
                const Acc v = h[c].get(i);
                squares += i >= k[c].skip ? v * v : (Acc)0;
                dot += i >= k[c].skip ? v * u[c].get(i) * w[c][i] : (Acc)0;
            }
        row_sums<LANES>(squares, dot);
        const Acc r = (Acc)1 / sqrt(squares / (Acc)a.D + (Acc)a.eps), back = dot * r * r / (Acc)a.D;
        const Acc counts = live ? r : (Acc)0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            Vec<IO, W> o;
            Vec<Stream, W> os;
#pragma unroll
            for (int i = 0; i < W; ++i) {
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
        __shared__ Acc sums[ROWS - 1][CH * W][LANES];
        if (threadIdx.x >= LANES) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < W; ++i) sums[threadIdx.x / LANES - 1][c * W + i][lane] = dw[c][i];
        }
        __syncthreads();
        if (threadIdx.x >= LANES) return;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int r = 0; r < ROWS - 1; ++r) dw[c][i] += sums[r][c * W + i][lane];
    }
    Acc *part = static_cast<Acc *>(a.partials) + (int64_t)blockIdx.x * a.D;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Vec<Acc, W> o;
#pragma unroll
        for (int i = 0; i < W; ++i) o.e[i] = dw[c][i];
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
        float power, rest;
        parts_of((float)r, &power, &rest);
        for (int64_t g = 0; g < a.groups; ++g) {
            const int64_t end = (g + 1) * group < a.D ? (g + 1) * group : a.D;
            float top = 0;
            for (int64_t i = g * group + threadIdx.x; i < end; i += RN_THREADS)
                top = larger(fabsf((float)value(i) * power * (float)weight(i)), top);
            top = row_max<RN_THREADS>(top);
            float lost = -INFINITY;
            for (int64_t i = g * group + threadIdx.x; i < end; i += RN_THREADS)
                lost = fmaxf(lost, lost_of((float)value(i) * power, (float)weight(i), top));
            lost = row_max<RN_THREADS>(lost);
            const float scale = scale_of(top, rest);
            if (threadIdx.x == 0) a.scales[row * a.groups + g] = scale;
            for (int64_t i = g * group + threadIdx.x; i < end; i += RN_THREADS) {
                const float h[1] = {(float)value(i) * power}, w[1] = {(float)weight(i)};
                float v[1];
                codes_of<1, true>(v, h, w, top, lost, rest, scale);
                static_cast<uint8_t *>(a.q)[base + i] = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v[0], 0.0f, 0, false) & 0xff);
            }
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

template <typename Stream> constexpr int chunk_of() { return sizeof(Stream) == 2 ? 8 : 4; }
constexpr int64_t WIDEST = 16384;        // columns of a row in registers
bool in_registers(int64_t D) { return D >= RN_WIDTH && D <= WIDEST; }
// Threads of a row (0: the kernels for any width), with chunks of one or two for each: lanes that have no columns cost as others do, and two
// chunks a thread are slower backward than one of twice as many threads.  bf16, forward and backward in us, the threads taken first:
//   65536 x 64    16: 10.2, 14.9   32: 14.8, 21.1            16384 x 1024   64: 26.5, 29.3   256: 26.9, 38.6
//   65536 x 128   16: 17.1, 16.5   32: 16.6, 20.7            16384 x 2048   256: 57.4, 59.2   512: 64.6, 72.1
//   32768 x 256   32: 16.6, 16.8   16: 15.9, 17.3   64: 16.6, 20.8   8192 x 4096   512: 55.2, 54.4   256: 55.6, 60.9   1024: 62.2, 83.3
//   32768 x 512   64: 27.5, 27.4   32: 26.3, 28.4            8192 x 8192    512: 106, 108   1024: 107, 122
int lanes_of(int64_t D) {
    return !in_registers(D) ? 0 : D <= 128 ? 16 : D <= 256 ? 32 : D <= 1024 ? 64 : D <= 2048 ? 256 : D <= 8192 ? 512 : 1024;
}
int64_t rows_of_group(int64_t D) { return lanes_of(D) == 0 ? 1 : threads_of(lanes_of(D)) / lanes_of(D); }
// Workgroups of the backward: one for each of the 256 CUs before any takes a second round of rows, then as many as are on the chip at
// once, with at least four rounds each, as every workgroup leaves a row of 32-bit sums; all with the same number of rounds.
int64_t backward_groups(int64_t N, int64_t D) {
    const int64_t rows = rows_of_group(D), rounds = (N + rows - 1) / rows;
    const int64_t most = 1024 * RN_THREADS / threads_of(lanes_of(D) ? lanes_of(D) : RN_THREADS);
    if (rounds <= 1024) return rounds < 256 ? rounds : 256;
    const int64_t each = rounds <= 4 * most ? 4 : (rounds + most - 1) / most;
    return (rounds + each - 1) / each;
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

// Rows `at` and the `n - 1` after them
template <typename IO, typename Stream> NormArgs rows_of(const NormArgs &a, int64_t at, int64_t n) {
    const auto moved = [](auto p, int64_t bytes) { return p == nullptr ? p : decltype(p)((uintptr_t)p + bytes); };
    NormArgs r = a;
    r.N = n;
    r.x = moved(a.x, at * a.D * sizeof(IO));
    r.res = moved(a.res, at * a.D * sizeof(Stream));
    r.y = moved(a.y, at * a.D * sizeof(IO));
    r.stored = moved(a.stored, at * a.D * sizeof(Stream));
    r.q = moved(a.q, at * a.D);
    r.scales = moved(a.scales, at * a.groups * sizeof(float));
    return r;
}

template <typename IO, typename Stream, bool FP8> int forward_of(const NormArgs &all, hipStream_t stream) {
    // A grid has less than 2^32 threads along an axis; of more the hardware starts the remainder, and no error comes.
    const int64_t per_group = rows_of_group(all.D), most = per_group * ((1ll << 31) / (lanes_of(all.D) ? threads_of(lanes_of(all.D)) : RN_THREADS));
    // 8 bits: a chunk is 8 columns in every type, as a group's chunks have to be in one wave
    constexpr int W = FP8 ? RN_WIDTH : chunk_of<Stream>(), PER = RN_WIDTH / W;
    for (int64_t at = 0; at < all.N; at += most) {
        const NormArgs a = rows_of<IO, Stream>(all, at, all.N - at < most ? all.N - at : most);
        const dim3 grid((unsigned)((a.N + per_group - 1) / per_group));
#define NORM_RUN(L, C) hipLaunchKernelGGL((norm_forward_kernel<IO, Stream, L, C * PER, W, FP8>), grid, threads, 0, stream, a)
        NORM_BY_WIDTH(NORM_RUN, hipLaunchKernelGGL((norm_forward_any_kernel<IO, Stream, FP8>), grid, threads, 0, stream, a));
#undef NORM_RUN
        const int rc = check_hip(hipGetLastError(), "norm_forward_kernel launch");
        if (rc) return rc;
    }
    return T2FW_OK;
}

template <typename IO, typename Stream> int backward_of(const NormArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    const int64_t groups = backward_groups(a.N, a.D), columns = (a.D + RW_COLUMNS - 1) / RW_COLUMNS;
    if (columns * RW_THREADS > 0xffffffffll) return fail(T2FW_ERR_BAD_SHAPE, "norm: too many columns for one launch of the weights' gradient");
    const dim3 grid((unsigned)groups);
    if (a.N > 0) {
        constexpr int W = chunk_of<Stream>(), PER = RN_WIDTH / W;
#define NORM_RUN(L, C) hipLaunchKernelGGL((norm_backward_kernel<IO, Stream, L, C * PER, W>), grid, threads, 0, stream, a)
        NORM_BY_WIDTH(NORM_RUN, hipLaunchKernelGGL((norm_backward_any_kernel<IO, Stream>), grid, threads, 0, stream, a));
#undef NORM_RUN
        const int rc = check_hip(hipGetLastError(), "norm_backward_kernel launch");
        if (rc) return rc;
    }
    hipLaunchKernelGGL((norm_weights_kernel<IO, Acc>), dim3((unsigned)columns), dim3(RW_THREADS), 0, stream, a, norm_partials(a.N, a.D));
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
