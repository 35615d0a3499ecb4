// The causal convolution of W = 2 to 8 taps per channel, z_t = bias + sum_j w_j xs_{t+j} with xs the W - 1 inputs before the sequence (the state)
// and its own, y = z or z sigmoid(z); what is before a selective scan.
//
// Bound by memory (1 x 32749 x 1021 float32 forward 50 us, 5.3 TB/s; 32 x 1024 x 4096 bf16 122 us forward, 4.4 TB/s, backward 208, 3.9): a lane owns
// 16 bytes of neighbouring channels of one row (backward: four channels) and 8 steps of them forward, so that an input is loaded once, and again from
// the cache for the lane that has the next steps.  A workgroup has 16 such lanes side by side (256 bytes of a step) and 16 stretches in time.
// Backward dx_p = sum_j w_j dz_{p+W-1-j} needs dz of the W - 1 steps after a lane's own too, which it makes again from x and the gradient: as many
// loads at once as there are, and no loop whose loads wait for the stores of the one before (stretches of 13 to 125 steps, dz handed on in registers: 41 us
// for 8 x 1024 x 1536 bf16, now 26).  The weights' gradients are summed in registers, over the stretches of a workgroup in
// shared memory, and over workgroups by a second launch: in a fixed order.
#include <type_traits>
#include "short_conv.hpp"
#include "activation.hpp"
#include "dies.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int THREADS = 256, R = 8;                              // R: steps of a lane
// ... backward: four where eight do not fit the registers of two waves
constexpr int back_steps(int taps, bool wide) { return taps + (wide ? 3 : 0) > 5 ? 4 : 8; }
constexpr int64_t MOST_GROUPS = (1ll << 32) / THREADS - 1;      // a grid has less than 2^32 threads along an axis

// Neighbouring blocks of channels of one die: where rows start anywhere they share lines (1 x 32749 x 1021 float32, forward and backward: 67 and 117 us, in runs of
// 16 50 and 102; 1536 channels of 16 bits, whose rows begin at whole lines, the same either way)
constexpr uint32_t NEAR = 16;

// Lanes side by side, workgroups side by side, stretches of a row, steps of one, workgroups one after another, rounds of stretches of one
struct ConvGrid {
    uint32_t lanes, per_row, blocks, stretches, steps, groups, rounds;
    bool fits;
};

__device__ __forceinline__ int64_t row_length(const ConvArgs &a, int64_t b) {
    if (a.lengths == nullptr) return a.T;
    const int64_t n = a.wide_lengths ? static_cast<const int64_t *>(a.lengths)[b] : static_cast<const int32_t *>(a.lengths)[b];
    return n < 0 ? 0 : n < a.T ? n : a.T;
}

template <typename IO, int VEC, int W> __device__ __forceinline__ void load_weights(float (&w)[VEC * W], const ConvArgs &a, int64_t d) {
    if (a.wide_w) {
        const Vec<float, VEC * W> v = load_vec<float, VEC * W>(static_cast<const float *>(a.w) + d * W);
#pragma unroll
        for (int i = 0; i < VEC * W; ++i) w[i] = v.e[i];
    } else {
        const Vec<IO, VEC * W> v = load_vec<IO, VEC * W>(static_cast<const IO *>(a.w) + d * W);
#pragma unroll
        for (int i = 0; i < VEC * W; ++i) w[i] = widen(v.e[i]);
    }
}
template <typename IO, int VEC> __device__ __forceinline__ void load_bias(float (&bias)[VEC], const ConvArgs &a, int64_t d) {
#pragma unroll
    for (int v = 0; v < VEC; ++v)
        bias[v] = a.bias == nullptr ? 0.0f : a.wide_w ? static_cast<const float *>(a.bias)[d + v] : widen(static_cast<const IO *>(a.bias)[d + v]);
}
template <typename IO, int VEC> __device__ __forceinline__ Vec<IO, VEC> nothing() {
    Vec<IO, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v.e[i] = narrow<IO>(0.0f);
    return v;
}
// The input at step p of a row, p >= -(W - 1); of a step beyond the last one that of the last (T > 0)
template <typename IO, int VEC, int W> __device__ __forceinline__ Vec<IO, VEC> input_at(const ConvArgs &a, int64_t b, int64_t p, int64_t d) {
    if (p < 0) {
        if (a.state == nullptr) return nothing<IO, VEC>();
        return load_vec<IO, VEC>(static_cast<const IO *>(a.state) + (b * (W - 1) + p + W - 1) * a.D + d);
    }
    return load_vec<IO, VEC>(static_cast<const IO *>(a.x) + b * a.x_b + (p < a.T ? p : a.T - 1) * a.x_t + d);
}

// Where a lane is: first channel, number of its stretch over all rows, row, first step
struct Place {
    int64_t d, q, b, t0;
    bool mine;
};
template <int VEC> __device__ __forceinline__ Place place_of(const ConvArgs &a, const ConvGrid &g, uint32_t round = 0) {
    Place p;
    const uint32_t piece = piece_of_work<NEAR>(), block = piece % g.blocks, group = piece / g.blocks, lane = threadIdx.x % g.lanes;
    const uint32_t slot = block * g.lanes + lane;
    p.q = ((int64_t)group * g.rounds + round) * (THREADS / g.lanes) + threadIdx.x / g.lanes;
    p.mine = slot < g.per_row && p.q < a.B * (int64_t)g.stretches;
    if (!p.mine) p.q = 0;
    p.b = (uint32_t)p.q / g.stretches;
    p.t0 = (p.q - p.b * g.stretches) * g.steps;
    const int64_t d = p.mine ? (int64_t)slot * VEC : 0;
    p.d = d + VEC <= a.D ? d : a.D - VEC;                // a row's last lane does channels of its neighbour again, to the same bits
    return p;
}

template <typename IO, int VEC, int W, bool SILU> __global__ __launch_bounds__(THREADS) void conv_forward_kernel(ConvArgs a, ConvGrid g) {
    constexpr bool FAST = sizeof(IO) == 2;
    const Place p = place_of<VEC>(a, g);
    if (!p.mine) return;
    const int64_t length = row_length(a, p.b);
    IO *const to = static_cast<IO *>(a.y) + (p.b * a.T + p.t0) * a.D + p.d;
    if (p.t0 >= length) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (p.t0 + r < a.T) store_vec(to + r * a.D, nothing<IO, VEC>());
    } else {
        Vec<IO, VEC> x[R + W - 1];
        if (p.t0 > 0) {
            const IO *at = static_cast<const IO *>(a.x) + p.b * a.x_b + (p.t0 - (W - 1)) * a.x_t + p.d;
            const int there = a.T - p.t0 < R ? (int)(a.T - p.t0) + W - 1 : R + W - 1;
#pragma unroll
            for (int i = 0; i < R + W - 1; ++i) {
                x[i] = load_vec<IO, VEC>(at);
                at += i + 1 < there ? a.x_t : 0;         // (of a step beyond the last one that again)
            }
        } else {
#pragma unroll
            for (int i = 0; i < R + W - 1; ++i) x[i] = input_at<IO, VEC, W>(a, p.b, i - (W - 1), p.d);
        }
        float w[VEC * W], bias[VEC];
        load_weights<IO, VEC, W>(w, a, p.d);
        load_bias<IO, VEC>(bias, a, p.d);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Vec<IO, VEC> y;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float z = bias[v];
#pragma unroll
                for (int j = 0; j < W; ++j) z = fmaf(w[v * W + j], widen(x[r + j].e[v]), z);
                y.e[v] = narrow<IO>(SILU ? silu_of<FAST>(z) : z);
            }
            if (p.t0 + r >= length) y = nothing<IO, VEC>();
            if (p.t0 + r < a.T) store_vec(to + r * a.D, y);
        }
    }
    if (p.t0 == 0) {
        IO *const last = static_cast<IO *>(a.last) + p.b * (W - 1) * a.D + p.d;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store_vec(last + j * a.D, input_at<IO, VEC, W>(a, p.b, length + j - (W - 1), p.d));
    }
}

// VEC elements as they came: 16-bit ones two to a register
template <typename IO, int VEC> struct Held {
    static constexpr int WORDS = (VEC * (int)sizeof(IO) + 3) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const IO *p) {
        w[WORDS - 1] = 0;
        __builtin_memcpy(w, p, VEC * sizeof(IO));
    }
    __device__ __forceinline__ void store(IO *p) const { __builtin_memcpy(p, w, VEC * sizeof(IO)); }
    __device__ __forceinline__ float get(int v) const { return element_of<IO>(w, v); }
    __device__ __forceinline__ void put(const float (&x)[VEC]) {
        IO e[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) e[v] = narrow<IO>(x[v]);
        w[WORDS - 1] = 0;
        __builtin_memcpy(w, e, sizeof(e));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0;
    }
};

// Two values per lane, added up over the halves of the wave (of 32 lanes) and of rows of 32 (of 16): the first in the lower, the second in the upper half
__device__ __forceinline__ float over_halves(float v0, float v1) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v0), __float_as_uint(v1), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float over_rows(float v0, float v1) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v0), __float_as_uint(v1), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename IO, int VEC, int W, bool SILU> __global__ __launch_bounds__(THREADS, 2) void conv_backward_kernel(ConvArgs a, ConvGrid g) {
    constexpr bool FAST = sizeof(IO) == 2;
    constexpr int SUMS = (VEC * (W + 1) + 3) / 4 * 4, LANES = 16, R = back_steps(W, sizeof(IO) == 4), H = W - 1;
    __shared__ float shares[THREADS / 64][SUMS][LANES];
    float sums[SUMS];                                    // of the weights and the bias of each channel
#pragma unroll
    for (int i = 0; i < SUMS; ++i) sums[i] = 0.0f;
    float w[VEC * W], bias[VEC];
    {
        const Place p = place_of<VEC>(a, g);
        load_weights<IO, VEC, W>(w, a, p.d);
        load_bias<IO, VEC>(bias, a, p.d);
    }
    IO *const d_state = static_cast<IO *>(a.d_state);
    const IO *const g_last = static_cast<const IO *>(a.g_last);
    for (uint32_t round = 0; round < g.rounds; ++round) {
        const Place p = place_of<VEC>(a, g, round);
        const int64_t length = p.mine ? row_length(a, p.b) : 0;
        IO *const d_x = static_cast<IO *>(a.d_x) + (p.b * a.T + p.t0) * a.D + p.d;
        if (p.mine && p.t0 < length) {
            const IO *xs = static_cast<const IO *>(a.x) + p.b * a.x_b + p.t0 * a.x_t + p.d, *gs = static_cast<const IO *>(a.g_y) + p.b * a.g_b + p.t0 * a.g_t + p.d;
            // steps t0 - H .. t0 + R + H of x, t0 .. t0 + R + H of the gradient
            Held<IO, VEC> x[R + 2 * H], gy[R + H];
            if (p.t0 >= H) {
                const IO *at = xs - H * a.x_t;
#pragma unroll
                for (int i = 0; i < H; ++i) x[i].load(at + i * a.x_t);
            } else {
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    const int64_t t = p.t0 - H + i;
                    x[i].clear();
                    if (t >= 0) x[i].load(xs + (i - H) * a.x_t);
                    else if (a.state != nullptr) x[i].load(static_cast<const IO *>(a.state) + (p.b * H + t + H) * a.D + p.d);
                }
            }
            const int there = a.T - p.t0 < R + H ? (int)(a.T - p.t0) : R + H, live = length - p.t0 < R + H ? (int)(length - p.t0) : R + H;
#pragma unroll
            for (int i = 0; i < R + H; ++i) {
                x[H + i].load(xs);
                gy[i].load(gs);
                xs += i + 1 < there ? a.x_t : 0;             // (of a step beyond the last one that again)
                gs += i + 1 < there ? a.g_t : 0;
            }
            const auto all = [&](auto WHOLE) {
                constexpr bool whole = decltype(WHOLE)::value;
                // what steps beyond the row's length hold does not count, whatever it is
                if constexpr (!whole) {
#pragma unroll
                    for (int i = 0; i < R + H; ++i)
                        if (i >= live) {
                            x[H + i].clear();
                            gy[i].clear();
                        }
                }
                // the gradient of the last inputs as they are handed on
                Held<IO, VEC> handed[R];
                if constexpr (!whole) {
#pragma unroll
                    for (int r = 0; r < R; ++r) handed[r].clear();
                    if (g_last != nullptr && p.t0 + R + H > length) {
                        const int64_t first = p.t0 - length + H;
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const int64_t at = first + r;
                            handed[r].load(g_last + (p.b * H + (at < 0 ? 0 : at < H ? at : H - 1)) * a.D + p.d);
                            if (at < 0 || at >= H) handed[r].clear();
                        }
                    }
                }
                float dz[R + H][VEC];
#pragma unroll
                for (int i = 0; i < R + H; ++i) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        float d = gy[i].get(v);
                        if constexpr (SILU) {
                            float z = bias[v];
#pragma unroll
                            for (int j = 0; j < W; ++j) z = fmaf(w[v * W + j], x[i + j].get(v), z);
                            d = d * silu_slope(z, sigmoid_of<FAST>(z));
                        }
                        dz[i][v] = whole || i < live ? d : 0.0f;
                        if (i < R) {                         // (the steps after the lane's own are others')
#pragma unroll
                            for (int j = 0; j < W; ++j) sums[v * (W + 1) + j] = fmaf(dz[i][v], x[i + j].get(v), sums[v * (W + 1) + j]);
                            sums[v * (W + 1) + W] += dz[i][v];
                        }
                    }
                    if (i < H) continue;
                    // all that counts for the input of W - 1 steps before
                    const int r = i - H;
                    const int64_t t = p.t0 + r;
                    float dx[VEC];
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        float d = 0.0f;
                        if constexpr (!whole) d = handed[r].get(v);
#pragma unroll
                        for (int j = 0; j < W; ++j) d = fmaf(w[v * W + j], dz[i - j][v], d);
                        dx[v] = whole || t < length ? d : 0.0f;
                    }
                    Held<IO, VEC> out;
                    out.put(dx);
                    if (whole || t < a.T) out.store(d_x + r * a.D);
                    // (one step after another: the registers of a step's numbers are free for the next one's)
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (p.t0 == 0 && d_state != nullptr) {
#pragma unroll
                    for (int m = 0; m < H; ++m) {
                        const int64_t at = m - length;
                        Held<IO, VEC> handed;
                        handed.clear();
                        if (g_last != nullptr && at >= 0) handed.load(g_last + (p.b * H + at) * a.D + p.d);
                        float ds[VEC];
#pragma unroll
                        for (int v = 0; v < VEC; ++v) {
                            ds[v] = handed.get(v);
#pragma unroll
                            for (int j = 0; j <= m; ++j) ds[v] = fmaf(w[v * W + j], dz[m - j][v], ds[v]);
                        }
                        Held<IO, VEC> out;
                        out.put(ds);
                        out.store(d_state + (p.b * H + m) * a.D + p.d);
                    }
                }
            };
            // nowhere in the wave the end of a row: neither what is beyond it nor what is handed on
            if (__all(live == R + H)) all(std::true_type{});
            else all(std::false_type{});
        } else if (p.mine) {
            Held<IO, VEC> none;
            none.clear();
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (p.t0 + r < a.T) none.store(d_x + r * a.D);
            if (p.t0 == 0 && d_state != nullptr) {           // a row without steps hands its state on
#pragma unroll
                for (int m = 0; m < H; ++m) {
                    Held<IO, VEC> handed;
                    handed.clear();
                    if (g_last != nullptr) handed.load(g_last + (p.b * H + m) * a.D + p.d);
                    handed.store(d_state + (p.b * H + m) * a.D + p.d);
                }
            }
        }
    }
    // Lanes of the same channels in a wave, then the waves.  Over the four rows of 16 lanes the values are spread while they are added.
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
    for (int i = 0; i < SUMS / 4; ++i) {
        float s = over_rows(over_halves(sums[i], sums[i + SUMS / 2]), over_halves(sums[i + SUMS / 4], sums[i + SUMS / 4 * 3]));
        for (uint32_t m = g.lanes; m < LANES; m <<= 1) s += __shfl_xor(s, m, 64);
        if (lane % LANES < (int)g.lanes) shares[wave][i + lane / 16 % 2 * (SUMS / 4) + lane / 32 * (SUMS / 2)][lane % LANES] = s;
    }
    __syncthreads();
    const uint32_t piece = piece_of_work<NEAR>(), block = piece % g.blocks, group = piece / g.blocks;
    constexpr int EACH = VEC * (W + 1);
    for (int i = threadIdx.x; i < (int)g.lanes * EACH; i += THREADS) {
        const int at = i % EACH, of = i / EACH;
        const int64_t slot = (int64_t)block * g.lanes + of, d = slot * VEC + VEC <= a.D ? slot * VEC : a.D - VEC;
        if (slot >= g.per_row) break;
        a.partials[((int64_t)group * a.D + d) * (W + 1) + at] = ((shares[0][at][of] + shares[1][at][of]) + shares[2][at][of]) + shares[3][at][of];
    }
}

// Sums over the workgroups: 64 columns of D (taps + 1) to a workgroup, four shares of the rows
template <typename IO> __global__ __launch_bounds__(THREADS) void conv_weights_kernel(ConvArgs a, int64_t rows) {
    __shared__ float parts[THREADS / 64][64];
    const int64_t width = a.D * (a.taps + 1), c = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int part = threadIdx.x / 64;
    float s = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (int64_t r = part; r < rows; r += THREADS / 64) s += a.partials[r * width + c];
    }
    parts[part][threadIdx.x % 64] = s;
    __syncthreads();
    if (part != 0 || c >= width) return;
    s = ((parts[0][threadIdx.x] + parts[1][threadIdx.x]) + parts[2][threadIdx.x]) + parts[3][threadIdx.x];
    const int64_t d = c / (a.taps + 1), j = c - d * (a.taps + 1);
    void *const to = j < a.taps ? a.d_w : a.d_bias;
    const int64_t at = j < a.taps ? d * a.taps + j : d;
    if (to == nullptr) return;
    if (a.wide_w) static_cast<float *>(to)[at] = s;
    else static_cast<IO *>(to)[at] = narrow<IO>(s);
}

// One token: y [B, D], the state one step on, in place or not.  A launch and a round to memory.
template <typename IO, int VEC, int W> __global__ __launch_bounds__(THREADS) void conv_step_kernel(ConvArgs a, uint32_t per_row, uint32_t n) {
    constexpr bool FAST = sizeof(IO) == 2;
    const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
    if (i >= n) return;
    const int64_t b = i / per_row, d0 = (int64_t)(i - (uint32_t)b * per_row) * VEC;
    // in place no channel may be done twice: the last lane of a row has what is left
    const int here = a.D - d0 < VEC ? (int)(a.D - d0) : VEC;
    const IO *const from = static_cast<const IO *>(a.state) + b * (W - 1) * a.D + d0, *const xp = static_cast<const IO *>(a.x) + b * a.x_b + d0;
    IO *const to = static_cast<IO *>(a.last) + b * (W - 1) * a.D + d0, *const yp = static_cast<IO *>(a.y) + b * a.D + d0;
    if (here == VEC) {
        Vec<IO, VEC> x[W], y;
        float w[VEC * W], bias[VEC];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) x[j] = load_vec<IO, VEC>(from + j * a.D);
        x[W - 1] = load_vec<IO, VEC>(xp);
        load_weights<IO, VEC, W>(w, a, d0);
        load_bias<IO, VEC>(bias, a, d0);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float z = bias[v];
#pragma unroll
            for (int j = 0; j < W; ++j) z = fmaf(w[v * W + j], widen(x[j].e[v]), z);
            y.e[v] = narrow<IO>(a.silu ? silu_of<FAST>(z) : z);
        }
        store_vec(yp, y);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store_vec(to + j * a.D, x[j + 1]);
        return;
    }
    for (int v = 0; v < here; ++v) {
        IO x[W];
        float w[W], bias[1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) x[j] = from[j * a.D + v];
        x[W - 1] = xp[v];
        load_weights<IO, 1, W>(w, a, d0 + v);
        load_bias<IO, 1>(bias, a, d0 + v);
        float z = bias[0];
#pragma unroll
        for (int j = 0; j < W; ++j) z = fmaf(w[j], widen(x[j]), z);
        yp[v] = narrow<IO>(a.silu ? silu_of<FAST>(z) : z);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) to[j * a.D + v] = x[j + 1];
    }
}

ConvGrid grid_of(int64_t B, int64_t T, int64_t D, int vec, int64_t steps, bool rounds = false) {
    ConvGrid g{};
    const int64_t per_row = (D + vec - 1) / vec;
    g.lanes = 16;
    while (g.lanes > 1 && g.lanes / 2 >= per_row) g.lanes /= 2;
    const int64_t blocks = (per_row + g.lanes - 1) / g.lanes, stretches = T <= 0 ? 1 : (T + steps - 1) / steps, TG = THREADS / g.lanes;
    const long double all = (long double)B * stretches;
    g.fits = per_row < 0x7fffffff && all < 0x7fffffff && (long double)blocks * ((all + TG - 1) / TG + 1) < MOST_GROUPS;
    g.per_row = (uint32_t)per_row;
    g.blocks = (uint32_t)blocks;
    g.stretches = (uint32_t)stretches;
    g.steps = (uint32_t)steps;
    g.groups = g.fits ? (uint32_t)((B * stretches + TG - 1) / TG) : 0;
    // Two workgroups for every CU, which load the weights and add their sums up once (backward, with the second launch: 8 x 1024 x 1536 bf16 34 us with a
    // workgroup for every 16 stretches, 26 so; 32 x 1024 x 4096 292 and 214)
    g.rounds = 1;
    if (rounds && g.groups > 0) {
        const int64_t n = blocks * g.groups / 512;
        g.rounds = n < 1 ? 1 : n < 16 ? (uint32_t)n : 16;
        g.groups = (g.groups + g.rounds - 1) / g.rounds;
    }
    return g;
}
ConvGrid backward_grid(int64_t B, int64_t T, int64_t D, int vec, int taps, bool wide) { return grid_of(B, T, D, vec, back_steps(taps, wide), true); }
// Channels of a lane: 16 bytes of them forward, four backward, where eight would take the registers of all waves but one
int vec_of(int64_t D, int dtype) {
    const int vec = dtype == T2FW_F32 ? 4 : 8;
    return D >= vec ? vec : 1;
}
int backward_vec_of(int64_t D) { return D >= 4 ? 4 : 1; }

template <typename IO, int VEC, int W> int launch_forward(const ConvArgs &a, const ConvGrid &g, hipStream_t stream) {
    if (a.silu) hipLaunchKernelGGL((conv_forward_kernel<IO, VEC, W, true>), dim3(g.blocks * g.groups), dim3(THREADS), 0, stream, a, g);
    else hipLaunchKernelGGL((conv_forward_kernel<IO, VEC, W, false>), dim3(g.blocks * g.groups), dim3(THREADS), 0, stream, a, g);
    return check_hip(hipGetLastError(), "conv_forward_kernel launch");
}
template <typename IO, int VEC, int W> int launch_backward(const ConvArgs &a, const ConvGrid &g, hipStream_t stream) {
    if (a.silu) hipLaunchKernelGGL((conv_backward_kernel<IO, VEC, W, true>), dim3(g.blocks * g.groups), dim3(THREADS), 0, stream, a, g);
    else hipLaunchKernelGGL((conv_backward_kernel<IO, VEC, W, false>), dim3(g.blocks * g.groups), dim3(THREADS), 0, stream, a, g);
    return check_hip(hipGetLastError(), "conv_backward_kernel launch");
}
template <typename IO, int VEC, int W> int launch_step(const ConvArgs &a, const ConvGrid &g, hipStream_t stream) {
    const uint32_t n = (uint32_t)(a.B * g.per_row);
    hipLaunchKernelGGL((conv_step_kernel<IO, VEC, W>), dim3((n + THREADS - 1) / THREADS), dim3(THREADS), 0, stream, a, g.per_row, n);
    return check_hip(hipGetLastError(), "conv_step_kernel launch");
}

int too_many() { return fail(T2FW_ERR_BAD_SHAPE, "short convolution: too many workgroups for one launch"); }

#define CONV_TAPS_OF(what, IO, VEC)                                  \
    switch (a.taps) {                                                \
        case 2: return what<IO, VEC, 2>(a, g, stream);               \
        case 3: return what<IO, VEC, 3>(a, g, stream);               \
        case 4: return what<IO, VEC, 4>(a, g, stream);               \
        case 5: return what<IO, VEC, 5>(a, g, stream);               \
        case 6: return what<IO, VEC, 6>(a, g, stream);               \
        case 7: return what<IO, VEC, 7>(a, g, stream);               \
        default: return what<IO, VEC, 8>(a, g, stream);              \
    }
#define CONV_OF(what, VEC16)                                                                                \
    template <typename IO, int VEC> int what##_taps(const ConvArgs &a, const ConvGrid &g, hipStream_t stream) { CONV_TAPS_OF(what, IO, VEC) } \
    int what##_of(const ConvArgs &a, const ConvGrid &g, int dtype, hipStream_t stream) {                    \
        const bool narrow_rows = a.D < (dtype == T2FW_F32 ? 4 : VEC16);                                     \
        switch (dtype) {                                                                                    \
            case T2FW_F32: return narrow_rows ? what##_taps<float, 1>(a, g, stream) : what##_taps<float, 4>(a, g, stream);       \
            case T2FW_F16: return narrow_rows ? what##_taps<_Float16, 1>(a, g, stream) : what##_taps<_Float16, VEC16>(a, g, stream); \
        }                                                                                                   \
        return narrow_rows ? what##_taps<__bf16, 1>(a, g, stream) : what##_taps<__bf16, VEC16>(a, g, stream);   \
    }
CONV_OF(launch_forward, 8)
CONV_OF(launch_backward, 4)
CONV_OF(launch_step, 8)

}  // namespace

int64_t conv_partials(int64_t B, int64_t T, int64_t D, int taps, int dtype) {
    return backward_grid(B, T, D, backward_vec_of(D), taps, dtype == T2FW_F32).groups;
}

int conv_forward(const ConvArgs &a, int dtype, hipStream_t stream) {
    const ConvGrid g = grid_of(a.B, a.T, a.D, vec_of(a.D, dtype), R);
    return g.fits ? launch_forward_of(a, g, dtype, stream) : too_many();
}

int conv_backward(const ConvArgs &a, int dtype, hipStream_t stream) {
    const ConvGrid g = backward_grid(a.B, a.T, a.D, backward_vec_of(a.D), a.taps, dtype == T2FW_F32);
    const int64_t columns = (a.D * (a.taps + 1) + 63) / 64;
    if (!g.fits || columns > MOST_GROUPS) return too_many();
    int rc = g.groups == 0 ? T2FW_OK : launch_backward_of(a, g, dtype, stream);
    if (rc) return rc;
    const dim3 grid((unsigned)columns), threads(THREADS);
    if (dtype == T2FW_F32) hipLaunchKernelGGL(conv_weights_kernel<float>, grid, threads, 0, stream, a, (int64_t)g.groups);
    else if (dtype == T2FW_F16) hipLaunchKernelGGL(conv_weights_kernel<_Float16>, grid, threads, 0, stream, a, (int64_t)g.groups);
    else hipLaunchKernelGGL(conv_weights_kernel<__bf16>, grid, threads, 0, stream, a, (int64_t)g.groups);
    return check_hip(hipGetLastError(), "conv_weights_kernel launch");
}

int conv_step(const ConvArgs &a, int dtype, hipStream_t stream) {
    const ConvGrid g = grid_of(a.B, 1, a.D, vec_of(a.D, dtype), R);
    return g.fits && a.B * (int64_t)g.per_row < 0x7fffffff ? launch_step_of(a, g, dtype, stream) : too_many();
}

}  // namespace t2fw
