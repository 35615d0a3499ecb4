// The selective scan, forward and single tokens.  select_tile.hpp has the layout and what bounds it.
#include <type_traits>
#include "select_tile.hpp"

namespace t2fw {
using namespace select_ns;
namespace {

template <typename IO, int G, bool GATED> __global__ __launch_bounds__(THREADS) void select_forward_kernel(SelectArgs a, Grid g) {
    constexpr int NP = G * S, Q = share<G>(), ROUNDS = TILE / Q;
    constexpr bool FAST = sizeof(IO) == 2;
    __shared__ float bs[2][TILE][NP], cs[2][TILE][NP];
    const Place p = place_of<G>(a, g);
    float rate[S], h[S] = {0.0f, 0.0f, 0.0f, 0.0f};
    load_rates(rate, a, p);
    const float bias = a.dt_bias == nullptr ? 0.0f : a.dt_bias[p.d], skip = a.skip == nullptr ? 0.0f : a.skip[p.d];
    const int tiles = (int)((p.live - p.begin + TILE - 1) / TILE);
    PerChannel<IO, G> x, dt, gate;
    PerStep<IO, G> b, c;
    const auto load = [&](int64_t t0) {
        x.load(a.x, a.x_b, a.x_t, a, p, t0);
        dt.load(a.dt, a.dt_b, a.dt_t, a, p, t0);
        if constexpr (GATED) gate.load(a.gate, a.z_b, a.z_t, a, p, t0);
        b.load(a.b, a.b_b, a.b_t, a, p, t0);
        c.load(a.c, a.c_b, a.c_t, a, p, t0);
    };
    if (tiles > 0) load(p.begin);
    at_chunk<G, false>(h, a, g, p, rate);
    for (int k = 0; k < tiles; ++k) {
        const int64_t t0 = p.begin + (int64_t)k * TILE;
        float (&b_here)[TILE][NP] = bs[k % 2], (&c_here)[TILE][NP] = cs[k % 2];
        b.store(&b_here[0][0], a, p, t0);
        c.store(&c_here[0][0], a, p, t0);
        if (a.ckpt != nullptr) {
            const Buffer at = result_of(a.ckpt + (p.b * g.tiles + t0 / TILE) * a.D * NP, a.D * NP * 4);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Four, Vec<float, S>{{h[0], h[1], h[2], h[3]}}), at, p.mine ? (uint32_t)((p.d * NP + p.n0) * 4) : BEYOND, 0, 0);
        }
        const Results<IO, G> y_to(a.y, a, p, t0);
        float length[ROUNDS], push[ROUNDS], add[ROUNDS], times[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool counts = t0 + r * Q + p.ng % Q < p.live;
            const float v = x.get(r), one = length_of<false>(a, dt.get(r) + bias).dt;
            length[r] = counts ? one : 0.0f;
            push[r] = counts ? one * v : 0.0f;
            add[r] = a.skip == nullptr ? 0.0f : skip * v;
            times[r] = 1.0f;
            if constexpr (GATED) times[r] = silu_of<FAST>(gate.get(r));
        }
        __syncthreads();
        load(k + 1 < tiles ? t0 + TILE : t0);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            float y[Q];
            const auto step = [&](auto J) {
                constexpr int j = decltype(J)::value;
                const float l = of_step<G, j>(length[r]), u = of_step<G, j>(push[r]);
                float bv[S], cv[S];
                load_padded(bv, &b_here[r * Q + j][p.n0]);
                load_padded(cv, &c_here[r * Q + j][p.n0]);
                y[j] = 0.0f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    h[s] = fmaf(exp2_of(l * rate[s]), h[s], u * bv[s]);
                    y[j] = fmaf(cv[s], h[s], y[j]);
                }
            };
            step(std::integral_constant<int, 0>{});
            if constexpr (Q >= 2) step(std::integral_constant<int, 1>{});
            if constexpr (Q == 4) { step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 3>{}); }
            const float out = (sum_steps<G>(y) + add[r]) * times[r];
            const int64_t t = t0 + r * Q + p.ng % Q;
            y_to.store(r, t < p.live ? out : 0.0f);
        }
    }
    // steps beyond the row's length
    for (int64_t t0 = p.begin + (int64_t)tiles * TILE; t0 < p.end; t0 += TILE) {
        const Results<IO, G> y_to(a.y, a, p, t0);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) y_to.store(r, 0.0f);
    }
    if (p.mine && p.chunk == g.chunks - 1) store_states(a.last + (p.b * a.D + p.d) * a.N, h, p.n0, a.N);
}

// One token: x, dt, gate, y [B, D], b, c [B, N]; the state in place or not.  A launch and a round to memory.
template <typename IO, int G> __global__ __launch_bounds__(THREADS) void select_step_kernel(SelectArgs a, uint32_t blocks) {
    constexpr bool FAST = sizeof(IO) == 2;
    const int64_t b = blockIdx.x / blocks, d = (int64_t)(blockIdx.x % blocks) * (THREADS / G) + threadIdx.x / G;
    const int n0 = threadIdx.x % G * S;
    const bool mine = d < a.D;
    float y = 0.0f, xv = 0.0f;
    if (mine) {
        float rate[S], h[S], bv[S], cv[S];
        const IO *const br = static_cast<const IO *>(a.b) + b * a.b_b, *const cr = static_cast<const IO *>(a.c) + b * a.c_b;
        // whole fours of states: one load each, at any address
        const bool fours = a.N % S == 0;
        if (fours && n0 < a.N) {
            load_padded(rate, a.a + d * a.N + n0);
            load_padded(h, a.s0 + (b * a.D + d) * a.N + n0);
            const Vec<IO, S> bs = load_vec<IO, S>(br + n0), cs = load_vec<IO, S>(cr + n0);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                bv[s] = widen(bs.e[s]);
                cv[s] = widen(cs.e[s]);
            }
        } else {
            load_states(rate, a.a + d * a.N, n0, a.N);
            load_states(h, a.s0 + (b * a.D + d) * a.N, n0, a.N);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                bv[s] = n0 + s < a.N ? widen(br[n0 + s]) : 0.0f;
                cv[s] = n0 + s < a.N ? widen(cr[n0 + s]) : 0.0f;
            }
        }
        xv = widen(static_cast<const IO *>(a.x)[b * a.x_b + d]);
        const float l = length_of<false>(a, widen(static_cast<const IO *>(a.dt)[b * a.dt_b + d]) + (a.dt_bias == nullptr ? 0.0f : a.dt_bias[d])).dt;
        const float u = l * xv;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            h[s] = fmaf(exp2_of(l * rate_of(rate[s])), h[s], u * bv[s]);
            y = fmaf(cv[s], h[s], y);
        }
        if (fours && n0 < a.N) store_padded(a.last + (b * a.D + d) * a.N + n0, h);
        else store_states(a.last + (b * a.D + d) * a.N, h, n0, a.N);
    }
    y = group_sum(y, G);
    if (!mine || n0 != 0) return;
    if (a.skip != nullptr) y = fmaf(a.skip[d], xv, y);
    if (a.gate != nullptr) y *= silu_of<FAST>(widen(static_cast<const IO *>(a.gate)[b * a.z_b + d]));
    static_cast<IO *>(a.y)[b * a.D + d] = narrow<IO>(y);
}

template <typename IO, int G> int launch_forward(const SelectArgs &a, const Grid &g, hipStream_t stream) {
    const unsigned row = (unsigned)(g.blocks * a.B);
    if (g.chunks > 1) {
        hipLaunchKernelGGL((select_maps_kernel<IO, G, false>), dim3(row * (g.chunks - 1)), dim3(THREADS), 0, stream, a, g);
        int rc = check_hip(hipGetLastError(), "select_maps_kernel launch");
        if (rc || (rc = launch_join<G, false>(a, g, stream))) return rc;
    }
    if (a.gate != nullptr) hipLaunchKernelGGL((select_forward_kernel<IO, G, true>), dim3(row * g.chunks), dim3(THREADS), 0, stream, a, g);
    else hipLaunchKernelGGL((select_forward_kernel<IO, G, false>), dim3(row * g.chunks), dim3(THREADS), 0, stream, a, g);
    return check_hip(hipGetLastError(), "select_forward_kernel launch");
}
template <typename IO, int G> int launch_step(const SelectArgs &a, uint32_t blocks, hipStream_t stream) {
    hipLaunchKernelGGL((select_step_kernel<IO, G>), dim3((unsigned)(a.B * blocks)), dim3(THREADS), 0, stream, a, blocks);
    return check_hip(hipGetLastError(), "select_step_kernel launch");
}

}  // namespace

int select_forward(const SelectArgs &a, int dtype, hipStream_t stream) {
    const Grid g = grid_of(a.B, a.T, a.D, a.N);
    if (!g.fits) return too_many();
    SELECT_OF(launch_forward, dtype, lanes_of(a.N), a, g, stream)
}

int select_step(const SelectArgs &a, int dtype, hipStream_t stream) {
    const Grid g = grid_of(a.B, 1, a.D, a.N);
    if (!g.fits) return too_many();
    SELECT_OF(launch_step, dtype, lanes_of(a.N), a, g.blocks, stream)
}

SelectPlan select_plan(int64_t B, int64_t T, int64_t D, int64_t N) {
    const Grid g = grid_of(B, T, D, N);
    const int64_t NP = lanes_of(N) * S;
    SelectPlan p{};
    if (!g.fits) return p;
    p.checkpoints = (size_t)(B * g.tiles * D * NP) * sizeof(float);
    p.forward = maps_bytes(g, B, D, N);
    p.backward = (maps_bytes(g, B, D, N) + 15) / 16 * 16 + (size_t)((int64_t)g.blocks * B * T * 2 * NP + (int64_t)g.chunks * B * D * (NP + 2)) * sizeof(float);
    return p;
}

}  // namespace t2fw
