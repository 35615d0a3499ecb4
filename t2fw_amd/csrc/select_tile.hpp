// What the selective scan's kernels share (select_fwd.hip, select_bwd.hip).
//
// h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t for every channel and state, y_t = <c_t, h_t> + skip x_t, out = y silu(gate).
//
// Layout: a lane owns four states of a channel, G = ceil(N / 4) lanes (a power of two) a channel, a workgroup of 256 threads 256 / G channels of one
// row and a chunk of its steps, which it goes through one by one with the states in registers.  What a step needs per channel (the step's length by the
// softplus, its product with the input, the gate) is made once, by one of the up to four lanes of a quad for each of as many steps, and
// handed to the others by the cross-lane moves that an instruction's operand can have.  b and c, the same for all channels, go through
// shared memory, 16 steps at a time.  Sums over a channel's lanes are made for as many steps as the quad has lanes at once.
//
// A stretch of steps is an affine map of the state before it, h -> exp(a sum dt) h + S: its decay needs no more than the sum of its steps' lengths.  So a
// sequence is cut in chunks where there are too few channels for the chip: one launch for the chunks' maps, and another in which a
// chunk puts those before it together and goes through its steps; of many chunks a launch between them puts the maps together.  It costs a chunk's
// decays twice.
//
// Bound by the vector units: a state and step is a product, an exponential (which takes two instructions' time), a product and two
// multiply-adds forward.
#pragma once
#include "activation.hpp"
#include "select.hpp"
#include "vec.hpp"

namespace t2fw {
namespace select_ns {

constexpr int THREADS = 256, S = 4, TILE = SELECT_TILE;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int64_t MOST_GROUPS = (1ll << 32) / THREADS - 1;      // a grid has less than 2^32 threads along an axis

// How a call is cut: channels of a workgroup are side by side, then rows, then chunks of `steps`
struct Grid {
    uint32_t blocks, chunks, tiles;      // tiles: of a whole row
    int64_t steps;
    bool joined;                         // many chunks: the states at their starts are made by a launch of their own
    bool fits;
};

// ---- a channel's lanes ---------------------------------------------------------------------------------------------
// steps that the lanes of a channel share out
template <int G> constexpr int share() { return G < 4 ? G : 4; }

// The value of the lane that has step j of a round
template <int G, int J> __device__ __forceinline__ float of_step(float v) {
    if constexpr (G == 1) return v;
    else if constexpr (G == 2) return dpp_move<J == 0 ? 0xA0 : 0xF5>(v);         // quad_perm [0,0,2,2], [1,1,3,3]
    else return dpp_move<J * 0x55>(v);                                           // quad_perm [J,J,J,J]
}
constexpr int DPP_ROW_SHL4 = 0x104, DPP_ROW_SHL8 = 0x108;

// Sums over the lanes of a channel, of one value per step of a round: the first lanes get that of their step each
template <int G> __device__ __forceinline__ float sum_steps(const float (&v)[share<G>()]) {
    if constexpr (G == 1) return v[0];
    const bool odd = threadIdx.x & 1;
    if constexpr (G == 2) {
        return (odd ? v[1] : v[0]) + dpp_move<DPP_QUAD_XOR1>(odd ? v[0] : v[1]);
    } else if constexpr (G >= 4) {
        const bool upper = threadIdx.x & 2;
        const float p = (odd ? v[1] : v[0]) + dpp_move<DPP_QUAD_XOR1>(odd ? v[0] : v[1]);
        const float q = (odd ? v[3] : v[2]) + dpp_move<DPP_QUAD_XOR1>(odd ? v[2] : v[3]);
        float r = (upper ? q : p) + dpp_move<DPP_QUAD_XOR2>(upper ? p : q);
        if constexpr (G >= 16) r += dpp_move<DPP_ROW_SHL8>(r);
        if constexpr (G >= 8) r += dpp_move<DPP_ROW_SHL4>(r);
        return r;
    }
}
// A sum over the steps of a round and all of them: over the lanes that have a step each
template <int G> __device__ __forceinline__ float sum_share(float v) { return group_sum(v, share<G>()); }

// ---- scalars of a step ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }

// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v|, and log(1 + e) = 2 artanh(r), r = e / (2 + e) <= 1/3: r + r^3 / 3 + ..., its seven terms off by 2^-26
// of it.  What the exponent's rounding leaves, up to 2^-18 of e at |v| = 80, is multiplied in: e^-|v| = 2^n e^(-|v| - n log 2) for n next to -|v| log2(e).  A
// step is off by 2^-20 of its length for v > -86; below that e comes to the smallest numbers, and is zero from -88 on.  (Four instructions: forward of
// 8 x 1024 x 1536 x 16 bf16 109 us without them, 111 so; of 4 x 1024 x 3000 x 4, where a lane makes every step of its channel, 57 and 59.)
struct Softplus {
    float value, slope;
};
template <bool SLOPE> __device__ __forceinline__ Softplus softplus_of(float v) {
    constexpr float LN2 = 0.69314718055994530942f;
    const float m = fmaxf(-fabsf(v), -128.0f), n = m * LOG2E, about = exp2_of(n);
    const float e = fmaf(about, fmaf(-n, LN2, m), about), r = e * __builtin_amdgcn_rcpf(2.0f + e), q = r * r;
    float p = 1.0f / 13.0f;
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = fmaf(p * q, r, r);
    Softplus s;
    s.value = fmaf(2.0f, p, v < 0.0f ? 0.0f : v);        // (NaN stays)
    s.slope = SLOPE ? (v >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e) : 0.0f;
    return s;
}

__device__ __forceinline__ int64_t row_length(const SelectArgs &a, int64_t b) {
    if (a.lengths == nullptr) return a.T;
    const int64_t n = a.wide_lengths ? static_cast<const int64_t *>(a.lengths)[b] : static_cast<const int32_t *>(a.lengths)[b];
    return n < 0 ? 0 : n < a.T ? n : a.T;
}

// Where a thread is
struct Place {
    int64_t b, d, begin, end, live;      // row, channel, first step of the chunk and the one after its last; ... after the last that counts
    int ng, n0;                          // lane of the channel, its first state
    uint32_t block, chunk;
    bool mine;                           // the channel exists (else it is the last one, and nothing of it is stored)
};
template <int G> __device__ __forceinline__ Place place_of(const SelectArgs &a, const Grid &g) {
    Place p;
    p.block = blockIdx.x % g.blocks;
    const uint32_t rest = blockIdx.x / g.blocks;
    p.b = rest % (uint32_t)a.B;
    p.chunk = rest / (uint32_t)a.B;
    p.ng = threadIdx.x % G;
    p.n0 = p.ng * S;
    p.d = (int64_t)p.block * (THREADS / G) + threadIdx.x / G;
    p.mine = p.d < a.D;
    if (!p.mine) p.d = a.D - 1;
    p.begin = p.chunk * g.steps;
    p.end = p.begin + g.steps < a.T ? p.begin + g.steps : a.T;
    const int64_t n = row_length(a, p.b);
    p.live = n < p.begin ? p.begin : n < p.end ? n : p.end;
    return p;
}

// A lane's states of [.., N] arrays; of those beyond N nothing
__device__ __forceinline__ void load_states(float (&v)[S], const float *at, int n0, int64_t N) {
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = n0 + s < N ? at[n0 + s] : 0.0f;
}
__device__ __forceinline__ void store_states(float *at, const float (&v)[S], int n0, int64_t N) {
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (n0 + s < N) at[n0 + s] = v[s];
}
__device__ __forceinline__ void load_padded(float (&v)[S], const float *at) {
    const Vec<float, S> x = load_vec<float, S>(at);
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = x.e[s];
}
__device__ __forceinline__ void store_padded(float *at, const float (&v)[S]) { store_vec(at, Vec<float, S>{{v[0], v[1], v[2], v[3]}}); }

// The decays' exponents per unit of step, for the hardware's exponential, which is that of two.  Finite, so that a step of no length (one that does not
// count) leaves every state as it is.
__device__ __forceinline__ float rate_of(float a) {
    const float r = a * LOG2E;
    return r < -3.4028234e38f ? -3.4028234e38f : r;
}
__device__ __forceinline__ void load_rates(float (&v)[S], const SelectArgs &a, const Place &p) {
    load_states(v, a.a + p.d * a.N, p.n0, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = rate_of(v[s]);
}

// Arrays through buffer descriptors: a scalar address for the tile, a lane's offset that stays as it is, and a scalar one for the round.  What is beyond the
// array is not loaded (zeros come) and not stored, so no branch stands between the accesses: with branches the compiler does not know
// how many are under way, and waits for the stores of a tile where it needs loads from before them (backward of 32 x 512 x 1536 x 16 bf16: 664 us, so
// 446; 412 with loads held as they come and no branch between the steps).
typedef __amdgpu_buffer_rsrc_t Buffer;
typedef uint32_t Four __attribute__((ext_vector_type(4)));
constexpr uint32_t BEYOND = 0x80000000u;                 // an offset that is in no array
__device__ __forceinline__ Buffer buffer_of(const void *at, int64_t bytes) {
    const int64_t n = bytes < 0 ? 0 : bytes < (int64_t)0xfffffff0u ? bytes : (int64_t)0xfffffff0u;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(at), 0, (int)(uint32_t)n, 0x00027000);
}
__device__ __forceinline__ Buffer result_of(void *at, int64_t bytes) { return buffer_of(at, bytes < (int64_t)BEYOND ? bytes : (int64_t)BEYOND); }
// An element on its way, in 32 bits: two of 16 bits would be put into one register, as soon as they are asked for, which waits for them
template <typename IO> __device__ __forceinline__ uint32_t load_from(Buffer b, uint32_t lane, uint32_t offset) {
    if constexpr (sizeof(IO) == 2) return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(b, lane, offset, 0);
    else return __builtin_amdgcn_raw_buffer_load_b32(b, lane, offset, 0);
}
template <typename IO> __device__ __forceinline__ float arrived(uint32_t v) { return element_of<IO>(&v, 0); }
template <typename IO> __device__ __forceinline__ void store_to(Buffer b, uint32_t lane, uint32_t offset, IO v) {
    if constexpr (sizeof(IO) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), b, lane, offset, 0);
    else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), b, lane, offset, 0);
}

// What a tile needs of the arrays, on its way: a lane's steps of those per channel ...
template <typename IO, int G> struct PerChannel {
    static constexpr int ROUNDS = TILE / share<G>();
    uint32_t v[ROUNDS];
    __device__ __forceinline__ float get(int r) const { return arrived<IO>(v[r]); }
    __device__ __forceinline__ void load(const void *base, int64_t row, int64_t step, const SelectArgs &a, const Place &p, int64_t t0) {
        const int64_t first = (int64_t)p.block * (THREADS / G);
        const IO *const at = static_cast<const IO *>(base) + p.b * row + t0 * step + first;
        const Buffer from = buffer_of(at, ((a.T - 1 - t0) * step + a.D - first) * (int64_t)sizeof(IO));
        const uint32_t lane = ((uint32_t)(p.ng % share<G>()) * (uint32_t)step + (uint32_t)(p.d - first)) * sizeof(IO);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) v[r] = load_from<IO>(from, lane, (uint32_t)(r * share<G>()) * (uint32_t)step * sizeof(IO));
    }
};
// ... and elements of b or c, which go to shared memory
template <typename IO, int G> struct PerStep {
    static constexpr int NP = G * S, EACH = (TILE * NP + THREADS - 1) / THREADS;
    uint32_t v[EACH];
    __device__ __forceinline__ void load(const void *base, int64_t row, int64_t step, const SelectArgs &a, const Place &p, int64_t t0) {
        const Buffer from = buffer_of(static_cast<const IO *>(base) + p.b * row + t0 * step, ((a.T - 1 - t0) * step + a.N) * (int64_t)sizeof(IO));
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int j = i * THREADS + threadIdx.x, n = j % NP;
            v[i] = load_from<IO>(from, j < TILE * NP && n < a.N ? ((uint32_t)(j / NP) * (uint32_t)step + n) * (uint32_t)sizeof(IO) : 0u, 0);
        }
    }
    // zeros for states that are none, and for steps that do not count, whatever they hold
    __device__ __forceinline__ void store(float *to, const SelectArgs &a, const Place &p, int64_t t0) const {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int j = i * THREADS + threadIdx.x;
            if (j < TILE * NP) to[j] = j % NP < a.N && t0 + j / NP < p.live ? arrived<IO>(v[i]) : 0.0f;
        }
    }
};
// Results per channel: a lane's steps of a tile
template <typename IO, int G> struct Results {
    Buffer to;
    uint32_t lane;
    int64_t D;
    __device__ __forceinline__ Results(void *base, const SelectArgs &a, const Place &p, int64_t t0) : D(a.D) {
        const int64_t first = (int64_t)p.block * (THREADS / G);
        to = result_of(static_cast<IO *>(base) + (p.b * a.T + t0) * a.D + first, ((a.T - t0) * a.D - first) * (int64_t)sizeof(IO));
        lane = p.mine && p.ng < share<G>() ? ((uint32_t)p.ng * (uint32_t)a.D + (uint32_t)(p.d - first)) * sizeof(IO) : BEYOND;
    }
    __device__ __forceinline__ void store(int r, float v) const {
        store_to<IO>(to, lane, (uint32_t)(r * share<G>()) * (uint32_t)D * sizeof(IO), narrow<IO>(v));
    }
};

// The state (BACK: the adjoint) at a chunk's start (end): the maps of the chunks before (after) it, from `first`
template <int G, bool BACK> __device__ __forceinline__ void through_maps(float (&h)[S], const SelectArgs &a, const Grid &g, const Place &p, const float (&rate)[S]) {
    constexpr int NP = G * S, AHEAD = 4;
    const int n = BACK ? (int)(g.chunks - 1 - p.chunk) : (int)p.chunk;
    const float *const maps = a.maps, *const lengths = a.maps + (int64_t)g.chunks * a.B * a.D * NP;
    for (int i = 0; i < n; i += AHEAD) {
        float v[AHEAD][S], sum[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int j = i + u < n ? i + u : n - 1, chunk = BACK ? (int)g.chunks - 1 - j : j;
            const int64_t at = ((int64_t)chunk * a.B + p.b) * a.D + p.d;
            load_padded(v[u], maps + at * NP + p.n0);
            sum[u] = lengths[at];
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (i + u < n) {
#pragma unroll
                for (int s = 0; s < S; ++s) h[s] = fmaf(exp2_of(rate[s] * sum[u]), h[s], v[u][s]);
            }
    }
}

// The state (BACK: the adjoint) at a chunk's start (end)
template <int G, bool BACK> __device__ __forceinline__ void at_chunk(float (&h)[S], const SelectArgs &a, const Grid &g, const Place &p, const float (&rate)[S]) {
    if (g.joined) {
        load_padded(h, a.maps + (((int64_t)p.chunk * a.B + p.b) * a.D + p.d) * (G * S) + p.n0);
        return;
    }
    const float *const first = BACK ? a.g_state : a.s0;
    if (first != nullptr) load_states(h, first + (p.b * a.D + p.d) * a.N, p.n0, a.N);
    through_maps<G, BACK>(h, a, g, p, rate);
}

// ... of all chunks, in place of their maps, where a chunk that goes through all the maps before it takes longer than the launch (forward and step of
// training in us, without it and with it: 8 x 1024 x 64 x 16 in 32 chunks 18, 50 and 19, 53; 8 x 2048 x 256 x 16 in 64 63, 192 and 59, 178; 1 x 16384
// x 64 x 16 in 512 120, 264 and 27, 78; 1 x 131072 x 64 x 16 in 1024 258, 652 and 91, 290).  JOIN_LANES lanes side by side in a workgroup, the chunks
// of each cut in JOIN_PARTS parts.  A thread puts the maps of its part together, the parts before it are put together in shared memory, in steps of
// twice as many, and it goes through its maps again.
template <int G, bool BACK, int JOIN_LANES> __global__ __launch_bounds__(THREADS) void select_join_kernel(SelectArgs a, Grid g) {
    constexpr int NP = G * S, AHEAD = 8, JOIN_PARTS = THREADS / JOIN_LANES;
    __shared__ float maps[2][S + 1][THREADS];
    const int part = threadIdx.x / JOIN_LANES;
    const int64_t lanes = a.B * a.D * G, unit = (int64_t)blockIdx.x * JOIN_LANES + threadIdx.x % JOIN_LANES;
    const bool mine = unit < lanes;
    const int64_t row = (mine ? unit : lanes - 1) / G, d = row % a.D;        // (row and channel)
    const int n0 = (int)((mine ? unit : lanes - 1) % G) * S;
    float *const states = a.maps + row * NP + n0;
    const float *const lengths = a.maps + (int64_t)g.chunks * a.B * a.D * NP + row;
    float rate[S], h[S] = {0.0f, 0.0f, 0.0f, 0.0f}, total = 0.0f;
    load_states(rate, a.a + d * a.N, n0, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) rate[s] = rate_of(rate[s]);
    // chunks in the order in which they follow; the last one's map is not needed
    const int chunks = (int)g.chunks, each = (chunks + JOIN_PARTS - 1) / JOIN_PARTS, begin = part * each, end = begin + each < chunks ? begin + each : chunks;
    const auto walk = [&](bool again) {
        for (int i = begin; i < end; i += AHEAD) {
            float v[AHEAD][S], sum[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int j = i + u < chunks - 1 ? i + u : chunks - 2;
                const int64_t at = (int64_t)(BACK ? chunks - 1 - j : j) * a.B * a.D;
                load_padded(v[u], states + at * NP);
                sum[u] = lengths[at];
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (i + u >= end) break;
                if (again && mine) store_padded(states + (int64_t)(BACK ? chunks - 1 - i - u : i + u) * a.B * a.D * NP, h);
                if (i + u == chunks - 1) break;
#pragma unroll
                for (int s = 0; s < S; ++s) h[s] = fmaf(exp2_of(rate[s] * sum[u]), h[s], v[u][s]);
                total += sum[u];
            }
        }
    };
    walk(false);
    int k = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) maps[0][s][threadIdx.x] = h[s];
    maps[0][S][threadIdx.x] = total;
    __syncthreads();
    for (int m = JOIN_LANES; m < THREADS; m *= 2, k ^= 1) {
        if ((int)threadIdx.x >= m) {
#pragma unroll
            for (int s = 0; s < S; ++s) h[s] = fmaf(exp2_of(rate[s] * total), maps[k][s][threadIdx.x - m], h[s]);
            total += maps[k][S][threadIdx.x - m];
        }
#pragma unroll
        for (int s = 0; s < S; ++s) maps[k ^ 1][s][threadIdx.x] = h[s];
        maps[k ^ 1][S][threadIdx.x] = total;
        __syncthreads();
    }
    // what is before the thread's part, on the state that is given
    const float *const given = BACK ? a.g_state : a.s0;
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = 0.0f;
    if (given != nullptr) load_states(h, given + row * a.N, n0, a.N);
    if (part > 0) {
        total = maps[k][S][threadIdx.x - JOIN_LANES];
#pragma unroll
        for (int s = 0; s < S; ++s) h[s] = fmaf(exp2_of(rate[s] * total), h[s], maps[k][s][threadIdx.x - JOIN_LANES]);
    }
    walk(true);
}

// A step's length, and its product with the input
template <bool SLOPE> struct StepLength {
    float dt, slope;
};
template <bool SLOPE> __device__ __forceinline__ StepLength<SLOPE> length_of(const SelectArgs &a, float raw) {
    if (!a.softplus) return {raw, 1.0f};
    const Softplus s = softplus_of<SLOPE>(raw);
    return {s.value, s.slope};
}

// The map of a chunk (BACK: of its adjoint): what it makes of a state of zero, and the sum of its steps' lengths
template <typename IO, int G, bool BACK> __global__ __launch_bounds__(THREADS) void select_maps_kernel(SelectArgs a, Grid g) {
    constexpr int NP = G * S, Q = share<G>(), ROUNDS = TILE / Q;
    constexpr bool FAST = sizeof(IO) == 2;
    __shared__ float rows[2][TILE][NP];
    // forward every chunk but the last, backward every one but the first
    Place p = place_of<G>(a, g);
    if (BACK) {
        p.chunk += 1;
        p.begin += g.steps;
        p.end = p.begin + g.steps < a.T ? p.begin + g.steps : a.T;
        const int64_t n = row_length(a, p.b);
        p.live = n < p.begin ? p.begin : n < p.end ? n : p.end;
    }
    float rate[S], h[S] = {0.0f, 0.0f, 0.0f, 0.0f}, total = 0.0f;
    load_rates(rate, a, p);
    const float bias = a.dt_bias == nullptr ? 0.0f : a.dt_bias[p.d];
    const int tiles = (int)((p.live - p.begin + TILE - 1) / TILE);
    PerChannel<IO, G> in, dt, gate;
    PerStep<IO, G> row;
    const auto load = [&](int k) {
        const int64_t t0 = p.begin + (int64_t)(BACK ? tiles - 1 - k : k) * TILE;
        in.load(BACK ? a.g_y : a.x, BACK ? a.g_b : a.x_b, BACK ? a.g_t : a.x_t, a, p, t0);
        dt.load(a.dt, a.dt_b, a.dt_t, a, p, t0);
        if (BACK && a.gate != nullptr) gate.load(a.gate, a.z_b, a.z_t, a, p, t0);
        row.load(BACK ? a.c : a.b, BACK ? a.c_b : a.b_b, BACK ? a.c_t : a.b_t, a, p, t0);
    };
    if (tiles > 0) load(0);
    for (int k = 0; k < tiles; ++k) {
        const int64_t t0 = p.begin + (int64_t)(BACK ? tiles - 1 - k : k) * TILE;
        float (&here)[TILE][NP] = rows[k % 2];
        row.store(&here[0][0], a, p, t0);
        float length[ROUNDS], push[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool counts = t0 + r * Q + p.ng % Q < p.live;
            const float raw = dt.get(r) + bias, one = length_of<false>(a, raw).dt;
            length[r] = counts ? one : 0.0f;
            float v = in.get(r);
            if (BACK && a.gate != nullptr) v *= silu_of<FAST>(gate.get(r));
            push[r] = counts ? (BACK ? v : one * v) : 0.0f;
            total += length[r];
        }
        __syncthreads();
        if (k + 1 < tiles) load(k + 1);
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int r = BACK ? ROUNDS - 1 - i : i;
            const auto step = [&](auto J) {
                constexpr int j = decltype(J)::value;
                const float l = of_step<G, j>(length[r]), u = of_step<G, j>(push[r]);
                float row_v[S];
                load_padded(row_v, &here[r * Q + j][p.n0]);
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const float decay = exp2_of(l * rate[s]);
                    h[s] = BACK ? decay * fmaf(u, row_v[s], h[s]) : fmaf(decay, h[s], u * row_v[s]);
                }
            };
            if constexpr (BACK) {
                if constexpr (Q == 4) { step(std::integral_constant<int, 3>{}); step(std::integral_constant<int, 2>{}); }
                if constexpr (Q >= 2) step(std::integral_constant<int, 1>{});
                step(std::integral_constant<int, 0>{});
            } else {
                step(std::integral_constant<int, 0>{});
                if constexpr (Q >= 2) step(std::integral_constant<int, 1>{});
                if constexpr (Q == 4) { step(std::integral_constant<int, 2>{}); step(std::integral_constant<int, 3>{}); }
            }
        }
    }
    total = sum_share<G>(total);
    if (!p.mine) return;
    const int64_t at = ((int64_t)p.chunk * a.B + p.b) * a.D + p.d;
    store_padded(a.maps + at * NP + p.n0, h);
    if (p.ng == 0) (a.maps + (int64_t)g.chunks * a.B * a.D * NP)[at] = total;
}

// ---- host ----------------------------------------------------------------------------------------------------------
inline int lanes_of(int64_t N) {
    int g = 1;
    while (g * S < N) g *= 2;
    return g;
}
// Chunks: the vector units of a CU are shared by its workgroups, so the time goes with the workgroups of the fullest CU times a chunk's tiles; half a
// workgroup and half a tile more stand for latencies that few workgroups do not hide, and for what a chunk takes whatever its length.  The maps cost
// 0.45 of the rest.  (D = 1536, N = 16 bf16, forward and step of training in us: 18 x 1024, 432 workgroups, whole 184 and 671, in two chunks 222 and 776;
// 14 x 1024 whole 182 and 661, in six 168 and 563; 8 x 1024 whole 134 and 490, in four 114 and 361, in eight 107 and 342, in 32 128 and 420; 8 x 128 whole
// 22 and 78, in four 23 and 74; 1 x 256 whole 37 and 129, in 16 15 and 41.  D = 64: 1 x 32 whole 8.6 and 27, in two 11 and 27.)
inline int64_t cost_of(int64_t rows, int64_t chunks, int64_t each) {
    const int64_t fullest = (rows * chunks + 255) / 256;
    return (2 * fullest + 1) * (2 * each + 1) * (chunks > 1 ? 29 : 20);
}
inline Grid grid_of(int64_t B, int64_t T, int64_t D, int64_t N) {
    Grid g{};
    const int64_t channels = THREADS / lanes_of(N), blocks = (D + channels - 1) / channels, tiles = T <= 0 ? 0 : (T + TILE - 1) / TILE;
    const long double rows = (long double)blocks * B;
    int64_t each = tiles == 0 ? 1 : tiles;
    if (rows > 0 && rows < 512 && tiles > 2) {
        const int64_t n = (int64_t)rows;
        int64_t least = cost_of(n, 1, each);
        for (int64_t full = 1; full <= 8; ++full) {
            const int64_t most = full * 256 / n, chunks = most < tiles ? most : tiles;
            if (chunks < 2) continue;
            const int64_t some = (tiles + chunks - 1) / chunks, cost = cost_of(n, (tiles + some - 1) / some, some);
            if (cost >= least) continue;              // (of equal ones the fewer: 8 x 4096 x 256 x 16 in 32 81 and 256, in 64 91 and 285)
            least = cost;
            each = some;
        }
    }
    g.steps = each * TILE;
    g.chunks = (uint32_t)(tiles == 0 ? 1 : (tiles + each - 1) / each);
    g.blocks = (uint32_t)blocks;
    g.joined = g.chunks > 48;
    g.fits = D < (1 << 21) &&      // (a step of the checkpoints is addressed by 32 bits)
             B < 0x7fffffff && tiles < 0x7fffffff && rows * g.chunks < MOST_GROUPS;
    g.tiles = (uint32_t)tiles;
    return g;
}
inline size_t maps_bytes(const Grid &g, int64_t B, int64_t D, int64_t N) {
    return g.chunks == 1 ? 0 : (size_t)g.chunks * B * D * (lanes_of(N) * S + 1) * sizeof(float);
}
template <int G, bool BACK> int launch_join(const SelectArgs &a, const Grid &g, hipStream_t stream) {
    if (!g.joined) return T2FW_OK;
    const int64_t lanes = a.B * a.D * G;
    // few parts where lanes alone make a workgroup for every CU (64 chunks of 1536 x 16 states 12.2 us in 64 parts, 7.3 in 16), else many (64 chunks of 64 x 16
    // states, with the scan, 15 us in 16, 14 in 64)
    if (g.chunks <= 128 && lanes >= 16 * 256) hipLaunchKernelGGL((select_join_kernel<G, BACK, 16>), dim3((unsigned)((lanes + 15) / 16)), dim3(THREADS), 0, stream, a, g);
    else hipLaunchKernelGGL((select_join_kernel<G, BACK, 4>), dim3((unsigned)((lanes + 3) / 4)), dim3(THREADS), 0, stream, a, g);
    return check_hip(hipGetLastError(), "select_join_kernel launch");
}
inline int too_many() { return fail(T2FW_ERR_BAD_SHAPE, "selective scan: too many channels, or workgroups for one launch"); }

#define SELECT_LANES(what, IO, lanes, ...)                                  \
    switch (lanes) {                                                        \
        case 1: return what<IO, 1>(__VA_ARGS__);                            \
        case 2: return what<IO, 2>(__VA_ARGS__);                            \
        case 4: return what<IO, 4>(__VA_ARGS__);                            \
        case 8: return what<IO, 8>(__VA_ARGS__);                            \
        default: return what<IO, 16>(__VA_ARGS__);                          \
    }
#define SELECT_OF(what, dtype, lanes, ...)                                  \
    switch (dtype) {                                                        \
        case T2FW_F32: SELECT_LANES(what, float, lanes, __VA_ARGS__)        \
        case T2FW_F16: SELECT_LANES(what, _Float16, lanes, __VA_ARGS__)     \
        default: SELECT_LANES(what, __bf16, lanes, __VA_ARGS__)             \
    }

}  // namespace select_ns
}  // namespace t2fw
