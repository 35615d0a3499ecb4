// The selective scan's gradients.  select_tile.hpp has the layout.
//
// With G_t the adjoint of h_t, G_t = dy_t c_t + exp(dt_{t+1} a) G_{t+1}, dy = g_y silu(gate), and p_t = G_t exp(dt_t a) h_{t-1}:
//   d_x = dt <G, b> + skip dy     d_dt = (<p, a> + x <G, b>) softplus'     d_gate = g_y y silu'(gate)     d_b = sum over channels of G dt x
//   d_c = sum over channels of dy h     d_a = sum over steps of p dt.
//
// The forward leaves the state before every 16 steps.  A workgroup goes through the tiles of its chunk from the last, each forward for the decays and
// states of its 16 steps, which stay in registers, and then back.  Sums over states are made as the forward's; sums over channels, two values per state
// and step: eight of a lane are spread over the wave while they are added (v_permlane swaps and masked row moves: two instructions for two
// values), then the waves are added in shared memory, and the blocks of channels by a second launch, as are the weights' gradients over rows and
// chunks: in a fixed order.
#include <type_traits>
#include "select_tile.hpp"

namespace t2fw {
using namespace select_ns;
namespace {

constexpr int DPP_ROW_ROR8 = 0x128;

// Two values per lane, added up over the halves of the wave (of 32 lanes) and of rows of 32 (of 16): the first value in the
// lower, the second in the upper half
__device__ __forceinline__ float over_halves(float v0, float v1) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v0), __float_as_uint(v1), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float over_rows(float v0, float v1) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v0), __float_as_uint(v1), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// ... of 8 lanes: masks of the banks that are written take the place of a choice
__device__ __forceinline__ float over_eights(float v0, float v1) {
    const float a = v0 + dpp_move<DPP_ROW_ROR8>(v0), b = v1 + dpp_move<DPP_ROW_ROR8>(v1);
    return threadIdx.x & 8 ? b : a;
}

// The value of the same lane of the other four in eight
__device__ __forceinline__ float other_fours(float v) {
    constexpr int SHL4 = 0x104, SHR4 = 0x114, EVEN = 0x5, ODD = 0xa;
    const int i = __float_as_int(v), up = __builtin_amdgcn_update_dpp(0, i, SHL4, 0xf, EVEN, true);
    return __int_as_float(__builtin_amdgcn_update_dpp(up, i, SHR4, 0xf, ODD, false));
}

// The sums over a wave's channels of a lane's four values for b and four for c, to the wave's place in shared memory
template <int G> __device__ __forceinline__ void add_channels(float *to, const float (&for_b)[S], const float (&for_c)[S]) {
    constexpr int NP = G * S;
    const int lane = threadIdx.x % 64;
    float r[S];
#pragma unroll
    for (int s = 0; s < S; ++s) r[s] = over_halves(for_b[s], for_c[s]);
    const float p0 = over_rows(r[0], r[2]), p1 = over_rows(r[1], r[3]);
    const int at = (lane / 32) * NP + lane % G * S + (lane / 16 % 2) * 2;
    if constexpr (G == 16) {
        to[at] = p0;
        to[at + 1] = p1;
    } else {
        // (lanes that hold the same sum write it to the same place: a choice of lanes would be a branch that no load is brought forward over)
        float v = over_eights(p0, p1);
        if constexpr (G <= 4) v += other_fours(v);
        if constexpr (G <= 2) v += dpp_move<DPP_QUAD_XOR2>(v);
        if constexpr (G <= 1) v += dpp_move<DPP_QUAD_XOR1>(v);
        to[at + (lane >> 3 & 1)] = v;
    }
}

template <typename IO, int G, bool GATED> __global__ __launch_bounds__(THREADS, G >= 4 ? 2 : 1) void select_backward_kernel(SelectArgs a, Grid g) {
    constexpr int NP = G * S, Q = share<G>(), ROUNDS = TILE / Q;
    constexpr bool FAST = sizeof(IO) == 2;
    __shared__ float bs[TILE][NP], cs[TILE][NP], sums[THREADS / 64][TILE][2 * NP];
    const Place p = place_of<G>(a, g);
    const int wave = threadIdx.x / 64;
    float rate[S], adj[S] = {0.0f, 0.0f, 0.0f, 0.0f}, d_a[S] = {0.0f, 0.0f, 0.0f, 0.0f}, d_skip = 0.0f, d_bias = 0.0f;
    load_rates(rate, a, p);
    const float bias = a.dt_bias == nullptr ? 0.0f : a.dt_bias[p.d], skip = a.skip == nullptr ? 0.0f : a.skip[p.d];
    const int tiles = (int)((p.live - p.begin + TILE - 1) / TILE);
    PerChannel<IO, G> x, dt, gate, gy;
    PerStep<IO, G> b, c;
    float next_h[S];
    const auto load = [&](int64_t t0) {
        x.load(a.x, a.x_b, a.x_t, a, p, t0);
        dt.load(a.dt, a.dt_b, a.dt_t, a, p, t0);
        if constexpr (GATED) gate.load(a.gate, a.z_b, a.z_t, a, p, t0);
        gy.load(a.g_y, a.g_b, a.g_t, a, p, t0);
        b.load(a.b, a.b_b, a.b_t, a, p, t0);
        c.load(a.c, a.c_b, a.c_t, a, p, t0);
        const Buffer at = buffer_of(a.ckpt + (p.b * g.tiles + t0 / TILE) * a.D * NP, a.D * NP * 4);
        const auto v = __builtin_bit_cast(Vec<float, S>, __builtin_amdgcn_raw_buffer_load_b128(at, (uint32_t)((p.d * NP + p.n0) * 4), 0, 0));
#pragma unroll
        for (int s = 0; s < S; ++s) next_h[s] = v.e[s];
    };
    if (tiles > 0) load(p.begin + (int64_t)(tiles - 1) * TILE);
    at_chunk<G, true>(adj, a, g, p, rate);
    // sums over the block's channels, of the tile
    const auto store_steps = [&](int64_t t0) {
        constexpr int ALL = TILE * 2 * NP;
        const Buffer to = result_of(a.bc + (((int64_t)p.block * a.B + p.b) * a.T + t0) * 2 * NP, (a.T - t0) * 2 * NP * 4);
#pragma unroll
        for (int i = 0; i < ALL; i += THREADS) {
            const int at = i + threadIdx.x, from = at < ALL ? at : 0;
            const float *const v = &sums[0][0][0] + from;
            store_to<float>(to, at < ALL ? at * 4u : BEYOND, 0, ((v[0] + v[ALL]) + v[2 * ALL]) + v[3 * ALL]);
        }
    };
    // steps beyond the row's length (those of b and c: select_steps_kernel)
    for (int64_t t0 = p.begin + (int64_t)tiles * TILE; t0 < p.end; t0 += TILE) {
        const Results<IO, G> d_x(a.d_x, a, p, t0), d_dt(a.d_dt, a, p, t0), d_gate(GATED ? a.d_gate : a.d_x, a, p, t0);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            d_x.store(r, 0.0f);
            d_dt.store(r, 0.0f);
            if constexpr (GATED) d_gate.store(r, 0.0f);
        }
    }
    for (int k = tiles - 1; k >= 0; --k) {
        const int64_t t0 = p.begin + (int64_t)k * TILE;
        const Results<IO, G> d_x(a.d_x, a, p, t0), d_dt(a.d_dt, a, p, t0), d_gate(GATED ? a.d_gate : a.d_x, a, p, t0);
        b.store(&bs[0][0], a, p, t0);
        c.store(&cs[0][0], a, p, t0);
        float length[ROUNDS], slope[ROUNDS], xs[ROUNDS], gys[ROUNDS], zs[ROUNDS], h0[S];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool counts = p.mine && t0 + r * Q + p.ng % Q < p.live;
            const auto one = length_of<true>(a, dt.get(r) + bias);
            length[r] = counts ? one.dt : 0.0f;
            slope[r] = counts ? one.slope : 0.0f;
            xs[r] = counts ? x.get(r) : 0.0f;
            gys[r] = counts ? gy.get(r) : 0.0f;
            zs[r] = GATED && counts ? gate.get(r) : 0.0f;
        }
#pragma unroll
        for (int s = 0; s < S; ++s) h0[s] = p.mine ? next_h[s] : 0.0f;
        __syncthreads();
        float decay[TILE][S], h[TILE][S], dy[ROUNDS], push[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            float y[Q];
            push[r] = length[r] * xs[r];
            const auto step = [&](auto J) {
                constexpr int j = decltype(J)::value;
                const int t = r * Q + j;
                const float l = of_step<G, j>(length[r]), u = of_step<G, j>(push[r]);
                float bv[S];
                load_padded(bv, &bs[t][p.n0]);
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    decay[t][s] = exp2_of(l * rate[s]);
                    h[t][s] = fmaf(decay[t][s], t > 0 ? h[t - 1][s] : h0[s], u * bv[s]);
                }
                if constexpr (GATED) {
                    float cv[S];
                    load_padded(cv, &cs[t][p.n0]);
                    y[j] = 0.0f;
#pragma unroll
                    for (int s = 0; s < S; ++s) y[j] = fmaf(cv[s], h[t][s], y[j]);
                }
            };
            step(std::integral_constant<int, 0>{});
            if constexpr (Q >= 2) step(std::integral_constant<int, 1>{});
            if constexpr (Q == 4) { step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 3>{}); }
            dy[r] = gys[r];
            if constexpr (GATED) {
                const float sig = sigmoid_of<FAST>(zs[r]), out = fmaf(skip, xs[r], sum_steps<G>(y));
                dy[r] = gys[r] * (zs[r] * sig);
                const int64_t t = t0 + r * Q + p.ng % Q;
                d_gate.store(r, t < p.live ? gys[r] * out * silu_slope(zs[r], sig) : 0.0f);
            }
        }
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int r = ROUNDS - 1 - i;
            // (when half of the decays and states are done with, whose registers it takes)
            if (i == ROUNDS / 2) load(k > 0 ? t0 - TILE : t0);
            float by_input[Q], by_decay[Q];
            const auto step = [&](auto J) {
                constexpr int j = decltype(J)::value;
                const int t = r * Q + j;
                const float l = of_step<G, j>(length[r]), u = of_step<G, j>(push[r]), d = of_step<G, j>(dy[r]);
                float bv[S], cv[S], for_b[S], for_c[S];
                load_padded(bv, &bs[t][p.n0]);
                load_padded(cv, &cs[t][p.n0]);
                by_input[j] = by_decay[j] = 0.0f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const float G_t = fmaf(cv[s], d, adj[s]);
                    by_input[j] = fmaf(G_t, bv[s], by_input[j]);
                    adj[s] = decay[t][s] * G_t;
                    const float q = adj[s] * (t > 0 ? h[t - 1][s] : h0[s]);
                    by_decay[j] = fmaf(q, rate[s], by_decay[j]);
                    d_a[s] = fmaf(q, l, d_a[s]);
                    for_b[s] = G_t * u;
                    for_c[s] = d * h[t][s];
                }
                add_channels<G>(sums[wave][t], for_b, for_c);
            };
            if constexpr (Q == 4) { step(std::integral_constant<int, 3>{}); step(std::integral_constant<int, 2>{}); }
            if constexpr (Q >= 2) step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 0>{});
            // (the rates are the logarithms of two of the decays)
            const float gb = sum_steps<G>(by_input), pa = sum_steps<G>(by_decay) * (1.0f / LOG2E);
            const float for_x = fmaf(length[r], gb, skip * dy[r]), for_dt = fmaf(xs[r], gb, pa) * slope[r];
            const int64_t t = t0 + r * Q + p.ng % Q;
            const bool counts = t < p.live;
            d_x.store(r, counts ? for_x : 0.0f);
            d_dt.store(r, counts ? for_dt : 0.0f);
            d_skip = fmaf(dy[r], xs[r], d_skip);
            d_bias += counts ? for_dt : 0.0f;
        }
        __syncthreads();
        store_steps(t0);
    }
    // (a channel's lanes beyond the first quad have the same steps as that)
    d_skip = sum_share<G>(d_skip);
    d_bias = sum_share<G>(d_bias);
    if (!p.mine) return;
    if (p.chunk == 0 && a.d_s0 != nullptr) store_states(a.d_s0 + (p.b * a.D + p.d) * a.N, adj, p.n0, a.N);
    float *const to = a.sums + (((int64_t)p.chunk * a.B + p.b) * a.D + p.d) * (NP + 2);
#pragma unroll
    for (int s = 0; s < S; ++s) to[p.n0 + s] = d_a[s];
    if (p.ng == 0) {
        to[NP] = d_skip;
        to[NP + 1] = d_bias;
    }
}

// Gradients of b and c: sums over the blocks of channels; zeros for steps that do not count, of which the blocks have left nothing, or, next to a state that is
// not finite, products of it with zero
template <typename IO> __global__ __launch_bounds__(THREADS) void select_steps_kernel(SelectArgs a, uint32_t blocks, int NP, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    if (i >= n) return;
    const int64_t t = i / (2 * NP);
    const int at = (int)(i - t * 2 * NP), s = at % NP;
    if (s >= a.N) return;
    const int64_t row = a.lengths == nullptr ? 0 : t / a.T;
    float v = 0.0f;
    if (a.lengths == nullptr || t - row * a.T < row_length(a, row)) {
#pragma unroll 8
        for (uint32_t k = 0; k < blocks; ++k) v += a.bc[k * n + i];
    }
    (at < NP ? static_cast<IO *>(a.d_b) : static_cast<IO *>(a.d_c))[t * a.N + s] = narrow<IO>(v);
}

// Gradients of a, skip and dt_bias: sums over rows and chunks, 64 columns to a workgroup, four shares of the rows
__global__ __launch_bounds__(THREADS) void select_weights_kernel(SelectArgs a, int NP, int64_t rows) {
    __shared__ float parts[THREADS / 64][64];
    const int64_t width = a.D * (NP + 2), i = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int part = threadIdx.x / 64;
    float v = 0.0f;
    if (i < width) {
#pragma unroll 8
        for (int64_t r = part; r < rows; r += THREADS / 64) v += a.sums[r * width + i];
    }
    parts[part][threadIdx.x % 64] = v;
    __syncthreads();
    if (part != 0 || i >= width) return;
    v = ((parts[0][threadIdx.x] + parts[1][threadIdx.x]) + parts[2][threadIdx.x]) + parts[3][threadIdx.x];
    const int64_t d = i / (NP + 2);
    const int at = (int)(i - d * (NP + 2));
    if (at < a.N) a.d_a[d * a.N + at] = v;
    if (at == NP && a.d_skip != nullptr) a.d_skip[d] = v;
    if (at == NP + 1 && a.d_bias != nullptr) a.d_bias[d] = v;
}

template <typename IO, int G> int launch_backward(const SelectArgs &a, const Grid &g, hipStream_t stream) {
    constexpr int NP = G * S;
    const unsigned row = (unsigned)(g.blocks * a.B);
    const int64_t n = a.B * a.T * 2 * NP, groups = (n + THREADS - 1) / THREADS, columns = (a.D * (NP + 2) + 63) / 64;
    if (groups > MOST_GROUPS || columns > MOST_GROUPS) return too_many();
    int rc;
    if (row > 0) {
        if (g.chunks > 1) {
            hipLaunchKernelGGL((select_maps_kernel<IO, G, true>), dim3(row * (g.chunks - 1)), dim3(THREADS), 0, stream, a, g);
            if ((rc = check_hip(hipGetLastError(), "select_maps_kernel launch")) || (rc = launch_join<G, true>(a, g, stream))) return rc;
        }
        if (a.gate != nullptr) hipLaunchKernelGGL((select_backward_kernel<IO, G, true>), dim3(row * g.chunks), dim3(THREADS), 0, stream, a, g);
        else hipLaunchKernelGGL((select_backward_kernel<IO, G, false>), dim3(row * g.chunks), dim3(THREADS), 0, stream, a, g);
        if ((rc = check_hip(hipGetLastError(), "select_backward_kernel launch"))) return rc;
    }
    if (n > 0) {
        hipLaunchKernelGGL((select_steps_kernel<IO>), dim3((unsigned)groups), dim3(THREADS), 0, stream, a, g.blocks, NP, n);
        if ((rc = check_hip(hipGetLastError(), "select_steps_kernel launch"))) return rc;
    }
    hipLaunchKernelGGL(select_weights_kernel, dim3((unsigned)columns), dim3(THREADS), 0, stream, a, NP, (int64_t)g.chunks * a.B);
    return check_hip(hipGetLastError(), "select_weights_kernel launch");
}

}  // namespace

int select_backward(const SelectArgs &args, int dtype, hipStream_t stream) {
    SelectArgs a = args;
    const Grid g = grid_of(a.B, a.T, a.D, a.N);
    if (!g.fits) return too_many();
    const int64_t NP = lanes_of(a.N) * S;
    // the scratch: maps, gradients of b and c by blocks, those of the weights by rows and chunks
    a.bc = a.maps + (maps_bytes(g, a.B, a.D, a.N) + 15) / 16 * 4;
    a.sums = a.bc + (int64_t)g.blocks * a.B * a.T * 2 * NP;
    SELECT_OF(launch_backward, dtype, lanes_of(a.N), a, g, stream)
}

}  // namespace t2fw
