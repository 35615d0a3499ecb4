// The recurrence with a vector for its state, h_t = f_t h_{t-1} + x_t per channel, over whole sequences.
//
// A stretch of steps is an affine map of the state before it, h -> P h + S with P the product of its gates, and maps of
// neighbouring stretches compose: (P2, S2) after (P1, S1) is (P2 P1, P2 S1 + S2).  The adjoint of the state runs the
// same way from the end, E_{t-1} = f_t (go_t + E_t), with d_x_t = go_t + E_t and d_f_t = d_x_t h_{t-1}.
//
// Layout: a lane owns 16 bytes of neighbouring channels of one row ("slot") and R consecutive steps of them, which it keeps
// in registers; a workgroup of 256 threads owns CL slots and TG = 256 / CL such stretches in a row, a chunk of
// C = TG R steps.  Slots are numbered over all rows of the batch, so that narrow rows share a workgroup.  Where the width is no
// multiple of the vector, a row's last slot starts early and does channels of its neighbour again, to the same bits.
//
// Every element is read once: a workgroup makes the map of its chunk, hands it to the chunks after it, and waits for theirs before it.
// A map travels as one 64-bit word (P, S), written and read atomically at the device's scope, in a place that a launch before has filled with a
// pattern that no map has; so the word says by itself whether it is there.  Chunks come in groups: the last one of a group
// also hands on the map of the whole group, and a chunk needs the groups before its own and the chunks before it in its
// group, about 2 sqrt(chunks) words.  They are composed in a fixed order, so the result does not depend on who is first.
// Chunks are numbered so that what a chunk waits for comes earlier in the grid, or among the same 128 workgroups.  Should the hardware not have
// started that workgroup all the same (another program on the device, say), a wait ends after a number of looks, and the workgroup makes
// the maps before its own itself from the inputs, by the same operations in the same order: every wait is bounded, and none needs
// another workgroup to run.
//
// Bound by memory where there is enough of it to move: 2 x 32768 x 1024 float32, GPU time, forward 149 us (805 MB, 5.4 TB/s), backward
// 243 us (1.34 GB, 5.5 TB/s; a copy of that size 5.0 to 5.4); 32 x 4096 x 1024 bf16 with logits 164 and 273 us (4.9 TB/s).  Two passes over the
// data, the chunks' maps first, took 338 and 805 us for the former.  Small calls are bound by the chain launch, load, hand on, wait, store:
// 1 x 8191 x 768 bf16 forward 14.8 us (11.4 in a variant that did not wait), 8 x 1024 x 768 forward 14.0, backward 16.1, and 2 for
// the launch that empties the words.
#include "gscan.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int GS_THREADS = 256;
constexpr int GS_CHANNELS = 64;          // channels of a workgroup (CHN below: 128 to FEW_STEPS of them where there are few steps)
constexpr int FEW_STEPS = 1024;
// A grid has less than 2^32 threads along an axis; of more the hardware starts the remainder, and no error comes
constexpr int64_t MOST_GROUPS = (1ll << 32) / GS_THREADS - 1;
constexpr int FEW_GROUPS = 2048;         // workgroups (the chip holds 512 to 1280 of them, by type and direction)

// elements of a lane: 32 in all, whatever the type
template <typename IO> struct Tile {
    static constexpr int VEC = 16 / sizeof(IO), R = 32 / VEC;
};
template <typename IO> struct AccT { using type = float; };
template <> struct AccT<double> { using type = double; };

template <typename Acc> struct Map {
    Acc p, s;
};

__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }
// m, and then n
template <typename Acc> __device__ __forceinline__ Map<Acc> after(const Map<Acc> &n, const Map<Acc> &m) {
    return {n.p * m.p, fused(n.p, m.s, n.s)};
}
// ... one step of gate g and input x more: h -> g h + x, or for the adjoint e -> g (e + x)
// (the same operations wherever it stands: no product of one step fused into the next)
template <bool BACK, typename Acc> __device__ __forceinline__ Map<Acc> extended(const Map<Acc> &m, Acc g, Acc x) {
#pragma clang fp contract(off)
    return {m.p * g, BACK ? g * (m.s + x) : fused(g, m.s, x)};
}

template <typename IO> __device__ __forceinline__ float gate_of(float z) {
    // From 16-bit logits: hardware exponential, off by |z| 1.25 2^-24 (its argument is rounded to 32 bits once multiplied by log2 e) and 2^-22, and
    // reciprocal, 2^-22: 2^-20 at z = -8, 2^-18 at -40.  The logit's own rounding to 16 bits is worth |z| 2^-12 or 2^-9.  From 32-bit ones: the library's,
    // with which 32 x 4096 x 1024 bf16 would take 258 and 401 us for 176 and 273.
    return sizeof(IO) == 2 ? __builtin_amdgcn_rcpf(1.0f + __expf(-z)) : 1.0f / (1.0f + expf(-z));
}
template <typename IO> __device__ __forceinline__ double gate_of(double z) { return 1.0 / (1.0 + exp(-z)); }
// f (1 - f) from the logit, without the cancellation in 1 - f
template <typename IO> __device__ __forceinline__ float gate_slope(float z) {
    if (sizeof(IO) == 2) {
        const float e = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
        return e * r * r;
    }
    const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
    return e * r * r;
}
template <typename IO> __device__ __forceinline__ double gate_slope(double z) {
    const double e = exp(-fabs(z)), r = 1.0 / (1.0 + e);
    return e * r * r;
}

// How a call is cut: slots of a row, workgroups side by side, chunks of the sequence, columns of one chunk in the scratch, chunks of a
// group, channels of a workgroup
struct GscanGrid {
    uint32_t per_row, blocks, chunks, group, channels;
    int64_t slots;
    bool fits;
};

__device__ __forceinline__ int64_t row_length(const GscanArgs &a, int64_t b) {
    if (a.lengths == nullptr) return a.T;
    const int64_t n = a.wide_lengths ? static_cast<const int64_t *>(a.lengths)[b] : static_cast<const int32_t *>(a.lengths)[b];
    return n < 0 ? 0 : n < a.T ? n : a.T;
}

// Where a lane's stretch is
template <int VEC, int R> struct Place {
    int64_t slot, b, d, t0;      // slot number, row, first channel, first step
    int steps;                   // steps within the tensor (0: nothing of this lane exists)
    int live;                    // ... and within the row's length
    int lane, group;             // slot within the workgroup, stretch within the chunk
    bool mine;
};
template <int VEC, int R, int CHN>
__device__ __forceinline__ Place<VEC, R> place_of(const GscanArgs &a, const GscanGrid &gr, int64_t block, int64_t chunk) {
    constexpr int CL = CHN / VEC, TG = GS_THREADS / CL;
    Place<VEC, R> p;
    p.lane = threadIdx.x % CL;
    p.group = threadIdx.x / CL;
    p.slot = block * CL + p.lane;
    p.mine = p.slot < a.B * (int64_t)gr.per_row;
    p.b = p.mine ? (uint32_t)p.slot / gr.per_row : 0;
    const int64_t d = (p.slot - p.b * gr.per_row) * VEC;
    p.d = d + VEC <= a.D ? d : a.D - VEC;
    p.t0 = chunk * (TG * R) + (int64_t)p.group * R;
    const int64_t length = row_length(a, p.b), left = p.mine ? a.T - p.t0 : 0, live = p.mine ? length - p.t0 : 0;
    p.steps = left < 0 ? 0 : left < R ? (int)left : R;
    p.live = live < 0 ? 0 : live < R ? (int)live : R;
    return p;
}

// A lane's vectors.  16-bit ones are held as they come, two to a register, and put together two at a time.
template <typename IO, int VEC> struct Held {
    static constexpr int PAIR = 1;
    Vec<IO, VEC> d;
    __device__ __forceinline__ void load(const IO *p) { d = load_vec<IO, VEC>(p); }
    __device__ __forceinline__ void store(IO *p) const { store_vec(p, d); }
    __device__ __forceinline__ auto get(int v) const { return widen(d.e[v]); }
    template <typename Acc> __device__ __forceinline__ void put(int v, const Acc (&x)[1]) { d.e[v] = narrow<IO>(x[0]); }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) d.e[v] = narrow<IO>(x);
    }
    __device__ __forceinline__ void as_it_came() {}      // 32-bit numbers take no more once they are made
};
template <typename IO> struct Held16 {
    static constexpr int PAIR = 2;
    Raw16 d;
    __device__ __forceinline__ void load(const IO *p) { d = load_raw(p); }
    __device__ __forceinline__ void store(IO *p) const { __builtin_memcpy(p, &d, sizeof(d)); }
    __device__ __forceinline__ float get(int v) const { return element<IO>(d, v); }
    __device__ __forceinline__ void put(int v, const float (&x)[2]) {
        const IO two[2] = {narrow<IO>(x[0]), narrow<IO>(x[1])};
        __builtin_memcpy(&d.w[v / 2], two, 4);
    }
    __device__ __forceinline__ void fill(float x) {
#pragma unroll
        for (int v = 0; v < 8; v += 2) put(v, {x, x});
    }
    // What has been made of it (32-bit numbers, gates) is made again from here on, rather than kept in two or four times the registers:
    // more workgroups on a CU, whose waits overlap (32 x 4096 x 1024 bf16 with logits: backward 311 us with the gates kept, 273 so).
    __device__ __forceinline__ void as_it_came() {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(d.w[i]));
    }
};
template <> struct Held<_Float16, 8> : Held16<_Float16> {};
template <> struct Held<__bf16, 8> : Held16<__bf16> {};

// Every load is made, whether its step counts or not (at a step that is there, or at the array's start), so that no branch stands between
// them and all are under way at once.
template <typename IO, int VEC, int R>
__device__ __forceinline__ void load_steps(Held<IO, VEC> (&v)[R], const void *base, int64_t row, int64_t step, const Place<VEC, R> &p) {
    const IO *at = static_cast<const IO *>(base);
    if (p.steps > 0) at += p.b * row + p.t0 * step + p.d;
    const int last = p.steps > 0 ? p.steps - 1 : 0;
#pragma unroll
    for (int r = 0; r < R; ++r) v[r].load(at + (r < last ? r : last) * step);
}
// What a step beyond the row's length holds does not count, whatever it is: it is taken as a gate of one (a logit of plus infinity) or an
// input of nothing, and its results are stored as zeros
template <typename IO, int VEC, int R> __device__ __forceinline__ void beyond_end(Held<IO, VEC> (&v)[R], const Place<VEC, R> &p, float with) {
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r >= p.live) v[r].fill(with);
}
template <typename IO, int VEC, int R>
__device__ __forceinline__ void store_steps(void *base, Held<IO, VEC> (&v)[R], int64_t D, int64_t T, const Place<VEC, R> &p) {
    IO *at = static_cast<IO *>(base) + (p.b * T + p.t0) * D + p.d;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= p.live) v[r].fill(0.0f);
        if (r < p.steps) v[r].store(at + r * D);
    }
}

template <typename IO, typename Acc, bool LOGITS, int VEC> __device__ __forceinline__ Acc gate_at(const Held<IO, VEC> &f, int v) {
    const Acc z = f.get(v);
    return LOGITS ? gate_of<IO>(z) : z;
}
constexpr float gate_beyond(bool logits) { return logits ? INFINITY : 1.0f; }

// The map of a channel over a stretch of gates g, forward in time, or of its adjoint, backward
template <typename IO, typename Acc, int VEC, int R, bool BACK>
__device__ __forceinline__ Map<Acc> fold_steps(const Acc (&g)[R], const Held<IO, VEC> (&x)[R], int v) {
    Map<Acc> m{1, 0};
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = BACK ? R - 1 - i : i;
        m = extended<BACK>(m, g[r], (Acc)x[r].get(v));
    }
    return m;
}

// Where a workgroup's channel is in [B, D] arrays; whether it is there
template <int VEC, int CHN> __device__ __forceinline__ bool channel_of(const GscanArgs &a, const GscanGrid &gr, int64_t block, int thread, int64_t *at) {
    const int64_t slot = block * (CHN / VEC) + thread / VEC, b = (uint32_t)slot / gr.per_row, d = (slot - b * gr.per_row) * VEC;
    *at = b * a.D + (d + VEC <= a.D ? d : a.D - VEC) + thread % VEC;
    return slot < a.B * (int64_t)gr.per_row;
}

// ---- maps from chunk to chunk --------------------------------------------------------------------------------------
constexpr uint64_t EMPTY = ~0ull;                        // a NaN of a pattern that word_of() gives to nothing
constexpr uint64_t NOTHING = 0x3f800000ull;              // the map that changes nothing
__device__ __forceinline__ uint64_t word_of(const Map<float> &m) {
    const uint64_t w = (uint64_t)__float_as_uint(m.s) << 32 | __float_as_uint(m.p);
    return w == EMPTY ? 0x7fc000007fc00000ull : w;       // another NaN
}
__device__ __forceinline__ Map<float> map_of(uint64_t w) { return {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))}; }
__device__ __forceinline__ void hand_on(uint64_t *word, const Map<float> &m) {
    __hip_atomic_store(word, word_of(m), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t look(const uint64_t *word) { return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The map of a whole chunk, by one wave, a channel for each lane: what its workgroup does, without it
template <typename IO, int VEC, int R, bool BACK, bool LOGITS>
__device__ __forceinline__ Map<float> map_alone(const GscanArgs &a, const GscanGrid &gr, int64_t block, int64_t chunk) {
    constexpr int TG = GS_THREADS / (GS_CHANNELS / VEC);
    const int lane = threadIdx.x % 64;
    const int64_t slot = block * (GS_CHANNELS / VEC) + lane / VEC;
    Map<float> all{1.0f, 0.0f};
    if (slot >= a.B * (int64_t)gr.per_row) return all;
    const int64_t b = (uint32_t)slot / gr.per_row, d0 = (slot - b * gr.per_row) * VEC, d = (d0 + VEC <= a.D ? d0 : a.D - VEC) + lane % VEC;
    const int64_t begin = (BACK ? gr.chunks - 1 - chunk : chunk) * (TG * R), end = row_length(a, b);
    const IO *f = static_cast<const IO *>(a.f) + b * a.f_b + d;
    const IO *x = BACK ? static_cast<const IO *>(a.g_out) + b * a.g_b + d : static_cast<const IO *>(a.x) + b * a.x_b + d;
    const int64_t x_t = BACK ? a.g_t : a.x_t;
    const auto gate = [&](int64_t t) {
        const float z = t < end ? (float)widen(f[t * a.f_t]) : 1.0f;
        return LOGITS && t < end ? gate_of<IO>(z) : z;
    };
    for (int i = 0; i < TG; ++i) {
        const int64_t t0 = begin + (BACK ? TG - 1 - i : i) * R;
        Map<float> m{1.0f, 0.0f};
        for (int k = 0; k < R; ++k) {
            const int64_t t = t0 + (BACK ? R - 1 - k : k);
            m.s = extended<BACK>(m, gate(t), t < end ? (float)widen(x[t * x_t]) : 0.0f).s;
        }
        for (int k = 0; k < R; ++k) m.p *= gate(t0 + k);             // (forward in time in either direction: the states' products)
        all = after(m, all);
    }
    return all;
}

// The maps lo, lo + 1, .. hi - 1 after one another, each waited for.  False: one did not come.
__device__ __forceinline__ bool wait_for(Map<float> &all, const uint64_t *words, int lo, int hi, int64_t slots, int looks) {
    constexpr int AHEAD = 8;
    const uint32_t lane = threadIdx.x % 64;
    all = {1.0f, 0.0f};
    for (int j = lo; j < hi; j += AHEAD) {
        uint64_t w[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) w[u] = j + u < hi ? look(words + (j + u) * slots + lane) : NOTHING;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            int left = looks;
            while (__any(w[u] == EMPTY)) {
                if (left-- <= 0) return false;
                __builtin_amdgcn_s_sleep(1);
                w[u] = look(words + (j + u) * slots + lane);
            }
            all = after(map_of(w[u]), all);
        }
    }
    return true;
}

// The recurrence's value before a chunk, in the threads of the first wave: `own` is the chunk's map there, `first` the value before the
// sequence; all threads of the workgroup call it.
template <typename IO, int VEC, int R, bool BACK, bool LOGITS>
__device__ __forceinline__ float value_before(const GscanArgs &a, const GscanGrid &gr, uint32_t block, uint32_t chunk, const Map<float> &own,
                                              float first) {
    if (gr.chunks == 1) return first;
    __shared__ Map<float> parts[GS_THREADS / 64][GS_CHANNELS];
    __shared__ bool missing[GS_THREADS / 64];
    uint64_t *const words = static_cast<uint64_t *>(a.words) + (int64_t)block * GS_CHANNELS, *const groups = words + gr.chunks * gr.slots;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    if (wave == 0 && chunk < gr.chunks - 1) hand_on(words + chunk * gr.slots + lane, own);
    // in the first group, four waves for the chunks before this one; later, two for the groups before this chunk's and two for the chunks
    // before it in its group
    const int group = chunk / gr.group, start = group * gr.group, c = (int)chunk;
    {
        const int lo = group == 0 ? c * wave / 4 : wave == 0 ? 0 : wave == 1 ? group / 2 : wave == 2 ? start : (start + c) / 2;
        const int hi = group == 0 ? c * (wave + 1) / 4 : wave == 0 ? group / 2 : wave == 1 ? group : wave == 2 ? (start + c) / 2 : c;
        Map<float> all;
        const bool came = wait_for(all, group != 0 && wave < 2 ? groups : words, lo, hi, gr.slots, a.looks);
        parts[wave][lane] = all;
        if (lane == 0) missing[wave] = !came;
    }
    __syncthreads();
    if (wave != 0) return 0.0f;
    if (__builtin_expect(missing[0] || missing[1] || missing[2] || missing[3], 0)) {
        // all of it from the inputs, put together as its workgroups do
        const Map<float> none{1.0f, 0.0f};
        Map<float> p[4] = {none, none, none, none}, q[4] = {none, none, none, none};
        const int last = gr.group - 1;
        for (int i = 0; i < c; ++i) {
            const Map<float> one = map_alone<IO, VEC, R, BACK, LOGITS>(a, gr, block, i);
            const int of = i / (int)gr.group, in = i - of * (int)gr.group, n = of == group ? c - start : last;       // chunks of its group that are put together
            const int part = of == 0 ? (in >= n / 4) + (in >= n * 2 / 4) + (in >= n * 3 / 4) : in < n / 2 ? 2 : 3;
            if (of < group && in == last) {
                const Map<float> whole = after(one, of == 0 ? after(q[3], after(q[2], after(q[1], q[0]))) : after(q[3], q[2]));
                if (of < group / 2) p[0] = after(whole, p[0]);
                else p[1] = after(whole, p[1]);
                q[0] = q[1] = q[2] = q[3] = none;
                continue;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (part == k) (of == group ? p : q)[k] = after(one, (of == group ? p : q)[k]);
        }
        for (int k = 0; k < 4; ++k) parts[k][lane] = p[k];
    }
    if (c == start + (int)gr.group - 1 && chunk < gr.chunks - 1) {
        Map<float> before = after(parts[3][lane], parts[2][lane]);
        if (group == 0) before = after(parts[3][lane], after(parts[2][lane], after(parts[1][lane], parts[0][lane])));
        hand_on(groups + group * gr.slots + lane, after(own, before));
    }
    float h = first;
#pragma unroll
    for (int i = 0; i < 4; ++i) h = fmaf(parts[i][lane].p, h, parts[i][lane].s);
    return h;
}

// double: every map is there from the launch before
template <typename IO, int VEC, int R, bool BACK, bool LOGITS>
__device__ __forceinline__ double value_before(const GscanArgs &a, const GscanGrid &gr, uint32_t block, uint32_t chunk, const Map<double> &,
                                               double first) {
    if (threadIdx.x >= GS_CHANNELS) return 0.0;
    const Map<double> *w = static_cast<const Map<double> *>(a.words) + (int64_t)block * GS_CHANNELS + threadIdx.x;
    for (int64_t c = 0; c < chunk; ++c) first = fma(w[c * gr.slots].p, first, w[c * gr.slots].s);
    return first;
}

// Before a call's main launch: the words empty
__global__ __launch_bounds__(GS_THREADS) void gscan_empty_kernel(uint64_t *words, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * GS_THREADS + threadIdx.x;
    if (i < n) words[i] = EMPTY;
}

// Which block of channels and which chunk (in the direction of the recurrence) a workgroup has.  The hardware deals workgroups out to the
// eight dies in turn, each with a cache of its own: runs of 16 neighbouring blocks go to one die, so that the lines that neighbours share,
// as they do where rows start anywhere, are fetched and written once (32 x 4096 bf16, forward: 1021 channels 250 -> 183 us, 1024
// 190 -> 163; in runs of 4 the backward of 32 x 4096 x 1024 takes 296 us, of 16 273).  Runs of 4 for few workgroups: a backward right after its
// forward, 8 x 1024 x 768, 15.9 us, of 16 18.3 (the same backward over and over does not tell them apart; 1 x 12000 x 1021 loses by it, 36.5 and
// 34.2).
constexpr uint32_t DIES = 8;
struct Turn {
    uint32_t block, chunk;
};
__device__ __forceinline__ Turn turn_of(const GscanGrid &gr) {
    const uint32_t near = gridDim.x < FEW_GROUPS ? 4 : 16, round = DIES * near;
    uint32_t n = blockIdx.x;
    if (n < gridDim.x / round * round) {
        const uint32_t in = n % round;
        n += in % DIES * near + in / DIES - in;
    }
    return {n % gr.blocks, n / gr.blocks};
}

// double: the map of every chunk but the last, for what comes after it in the direction of the recurrence
template <typename IO, typename Acc, int VEC, int R, bool BACK, bool LOGITS>
__global__ __launch_bounds__(GS_THREADS) void gscan_maps_kernel(GscanArgs a, GscanGrid gr) {
    constexpr int CL = GS_CHANNELS / VEC, TG = GS_THREADS / CL;
    __shared__ Map<Acc> maps[TG][GS_CHANNELS];
    const uint32_t block = blockIdx.x % gr.blocks, chunk = blockIdx.x / gr.blocks;
    const Place<VEC, R> p = place_of<VEC, R, GS_CHANNELS>(a, gr, block, BACK ? gr.chunks - 1 - chunk : chunk);
    Held<IO, VEC> x[R], f[R];
    load_steps<IO, VEC, R>(f, a.f, a.f_b, a.f_t, p);
    load_steps<IO, VEC, R>(x, BACK ? a.g_out : a.x, BACK ? a.g_b : a.x_b, BACK ? a.g_t : a.x_t, p);
    beyond_end<IO, VEC, R>(f, p, gate_beyond(LOGITS));
    beyond_end<IO, VEC, R>(x, p, 0.0f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Acc g[R];
#pragma unroll
        for (int r = 0; r < R; ++r) g[r] = gate_at<IO, Acc, LOGITS>(f[r], v);
        maps[p.group][p.lane * VEC + v] = fold_steps<IO, Acc, VEC, R, BACK>(g, x, v);
    }
    __syncthreads();
    if (threadIdx.x >= GS_CHANNELS) return;
    Map<Acc> all{1, 0};
#pragma unroll
    for (int i = 0; i < TG; ++i) all = after(maps[BACK ? TG - 1 - i : i][threadIdx.x], all);
    static_cast<Map<Acc> *>(a.words)[chunk * gr.slots + (int64_t)block * GS_CHANNELS + threadIdx.x] = all;
}

template <typename IO, typename Acc, int VEC, int R, int CHN, bool LOGITS>
__global__ __launch_bounds__(GS_THREADS, sizeof(Acc) == 8 ? 1 : sizeof(IO) == 2 ? 5 : 4) void gscan_forward_kernel(GscanArgs a, GscanGrid gr) {
    constexpr int CL = CHN / VEC, TG = GS_THREADS / CL, PAIR = Held<IO, VEC>::PAIR;
    __shared__ Map<Acc> maps[TG][CHN];
    const Turn turn = turn_of(gr);
    const uint32_t block = turn.block, chunk = turn.chunk;
    const Place<VEC, R> p = place_of<VEC, R, CHN>(a, gr, block, chunk);
    int64_t at = 0;
    const bool first = CHN == GS_CHANNELS && threadIdx.x < GS_CHANNELS, there = first && channel_of<VEC, CHN>(a, gr, block, threadIdx.x, &at);
    Acc h = there && a.s0 != nullptr ? static_cast<const Acc *>(a.s0)[at] : (Acc)0;
    Held<IO, VEC> x[R], f[R];
    load_steps<IO, VEC, R>(f, a.f, a.f_b, a.f_t, p);
    load_steps<IO, VEC, R>(x, a.x, a.x_b, a.x_t, p);
    beyond_end<IO, VEC, R>(f, p, gate_beyond(LOGITS));
    beyond_end<IO, VEC, R>(x, p, 0.0f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Acc g[R];
#pragma unroll
        for (int r = 0; r < R; ++r) g[r] = gate_at<IO, Acc, LOGITS>(f[r], v);
        maps[p.group][p.lane * VEC + v] = fold_steps<IO, Acc, VEC, R, false>(g, x, v);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        x[r].as_it_came();
        f[r].as_it_came();
    }
    __syncthreads();
    if constexpr (CHN == GS_CHANNELS) {
        Map<Acc> own{1, 0};
        if (first) {
#pragma unroll 8
            for (int i = 0; i < TG; ++i) own = after(maps[i][threadIdx.x], own);
        }
        h = value_before<IO, VEC, R, false, LOGITS>(a, gr, block, chunk, own, h);
        if (first) {
            if (a.ckpt != nullptr) static_cast<Acc *>(a.ckpt)[chunk * gr.slots + (int64_t)block * GS_CHANNELS + threadIdx.x] = h;
#pragma unroll 8
            for (int i = 0; i < TG; ++i) {
                const Map<Acc> m = maps[i][threadIdx.x];
                maps[i][threadIdx.x].s = h;              // the state before this stretch
                h = m.p * h + m.s;
            }
            if (there && chunk == gr.chunks - 1) static_cast<Acc *>(a.final_state)[at] = h;
        }
    } else {
        // a chunk that is the whole sequence
        for (int column = threadIdx.x; column < CHN; column += GS_THREADS) {
            const bool is = channel_of<VEC, CHN>(a, gr, block, column, &at);
            Acc h = is && a.s0 != nullptr ? static_cast<const Acc *>(a.s0)[at] : (Acc)0;
            if (a.ckpt != nullptr) static_cast<Acc *>(a.ckpt)[(int64_t)block * CHN + column] = h;
#pragma unroll
            for (int i = 0; i < TG; ++i) {
                const Map<Acc> m = maps[i][column];
                maps[i][column].s = h;
                h = m.p * h + m.s;
            }
            if (is) static_cast<Acc *>(a.final_state)[at] = h;
        }
    }
    __syncthreads();
    // the results take their inputs' registers
#pragma unroll
    for (int v = 0; v < VEC; v += PAIR) {
        Acc s[PAIR];
#pragma unroll
        for (int j = 0; j < PAIR; ++j) s[j] = maps[p.group][p.lane * VEC + v + j].s;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Acc out[PAIR];
#pragma unroll
            for (int j = 0; j < PAIR; ++j) {
                s[j] = fused(gate_at<IO, Acc, LOGITS>(f[r], v + j), s[j], (Acc)x[r].get(v + j));
                out[j] = s[j];
            }
            x[r].put(v, out);
        }
    }
    store_steps<IO, VEC, R>(a.out, x, a.D, a.T, p);
}

template <typename IO, typename Acc, int VEC, int R, int CHN, bool LOGITS>
__global__ __launch_bounds__(GS_THREADS, sizeof(Acc) == 8 ? 1 : sizeof(IO) == 2 ? 4 : 2) void gscan_backward_kernel(GscanArgs a, GscanGrid gr) {
    constexpr int CL = CHN / VEC, TG = GS_THREADS / CL, PAIR = Held<IO, VEC>::PAIR;
    __shared__ Map<Acc> maps[TG][CHN];                   // states: forward in time
    __shared__ Acc sums[TG][CHN];                        // adjoints: backward, with the same gate products
    const Turn turn = turn_of(gr);
    const uint32_t block = turn.block, from_end = turn.chunk, chunk = gr.chunks - 1 - from_end;
    const Place<VEC, R> p = place_of<VEC, R, CHN>(a, gr, block, chunk);
    int64_t at = 0;
    const bool first = CHN == GS_CHANNELS && threadIdx.x < GS_CHANNELS, there = first && channel_of<VEC, CHN>(a, gr, block, threadIdx.x, &at);
    Acc e = there && a.g_state != nullptr ? static_cast<const Acc *>(a.g_state)[at] : (Acc)0;
    Acc h = first ? static_cast<const Acc *>(a.ckpt)[chunk * gr.slots + (int64_t)block * GS_CHANNELS + threadIdx.x] : (Acc)0;
    Held<IO, VEC> x[R], f[R], go[R];
    load_steps<IO, VEC, R>(f, a.f, a.f_b, a.f_t, p);
    load_steps<IO, VEC, R>(go, a.g_out, a.g_b, a.g_t, p);
    load_steps<IO, VEC, R>(x, a.x, a.x_b, a.x_t, p);
    beyond_end<IO, VEC, R>(f, p, gate_beyond(LOGITS));
    beyond_end<IO, VEC, R>(go, p, 0.0f);
    beyond_end<IO, VEC, R>(x, p, 0.0f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Acc g[R];
#pragma unroll
        for (int r = 0; r < R; ++r) g[r] = gate_at<IO, Acc, LOGITS>(f[r], v);
        maps[p.group][p.lane * VEC + v] = fold_steps<IO, Acc, VEC, R, false>(g, x, v);
        sums[p.group][p.lane * VEC + v] = fold_steps<IO, Acc, VEC, R, true>(g, go, v).s;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        x[r].as_it_came();
        f[r].as_it_came();
        go[r].as_it_came();
    }
    __syncthreads();
    if constexpr (CHN == GS_CHANNELS) {
        Map<Acc> own{1, 0};
        if (first) {
#pragma unroll 8
            for (int i = TG - 1; i >= 0; --i) own = after({maps[i][threadIdx.x].p, sums[i][threadIdx.x]}, own);
        }
        e = value_before<IO, VEC, R, true, LOGITS>(a, gr, block, from_end, own, e);
        if (first) {
#pragma unroll 8
            for (int i = 0; i < TG; ++i) {
                const Map<Acc> m = maps[i][threadIdx.x];
                maps[i][threadIdx.x].s = h;              // the state before this stretch
                h = m.p * h + m.s;
            }
#pragma unroll 8
            for (int i = TG - 1; i >= 0; --i) {
                const Acc pr = maps[i][threadIdx.x].p, s = sums[i][threadIdx.x];
                sums[i][threadIdx.x] = e;                // the adjoint after it
                e = pr * e + s;
            }
            if (there && chunk == 0 && a.d_s0 != nullptr) static_cast<Acc *>(a.d_s0)[at] = e;
        }
    } else {
        for (int column = threadIdx.x; column < CHN; column += GS_THREADS) {
            const bool is = channel_of<VEC, CHN>(a, gr, block, column, &at);
            Acc e = is && a.g_state != nullptr ? static_cast<const Acc *>(a.g_state)[at] : (Acc)0;
            Acc h = static_cast<const Acc *>(a.ckpt)[(int64_t)block * CHN + column];
#pragma unroll
            for (int i = 0; i < TG; ++i) {
                const Map<Acc> m = maps[i][column];
                maps[i][column].s = h;
                h = m.p * h + m.s;
            }
#pragma unroll
            for (int i = TG - 1; i >= 0; --i) {
                const Acc pr = maps[i][column].p, s = sums[i][column];
                sums[i][column] = e;
                e = pr * e + s;
            }
            if (is && a.d_s0 != nullptr) static_cast<Acc *>(a.d_s0)[at] = e;
        }
    }
    __syncthreads();
    // the results take their inputs' registers
#pragma unroll
    for (int v = 0; v < VEC; v += PAIR) {
        Acc before[R][PAIR], g[R][PAIR], later[PAIR];
#pragma unroll
        for (int j = 0; j < PAIR; ++j) {
            Acc h = maps[p.group][p.lane * VEC + v + j].s;
            later[j] = sums[p.group][p.lane * VEC + v + j];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                g[r][j] = gate_at<IO, Acc, LOGITS>(f[r], v + j);
                before[r][j] = h;
                h = fused(g[r][j], h, (Acc)x[r].get(v + j));
            }
        }
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            Acc dx[PAIR], df[PAIR];
#pragma unroll
            for (int j = 0; j < PAIR; ++j) {
                const Acc d = (Acc)go[r].get(v + j) + later[j];
                later[j] = g[r][j] * d;
                const Acc slope = LOGITS ? (Acc)gate_slope<IO>((Acc)f[r].get(v + j)) : (Acc)1;
                dx[j] = d;
                df[j] = d * before[r][j] * slope;
            }
            go[r].put(v, dx);
            x[r].put(v, df);
        }
    }
    store_steps<IO, VEC, R>(a.d_x, go, a.D, a.T, p);
    store_steps<IO, VEC, R>(a.d_f, x, a.D, a.T, p);
}

// No steps: the value before them (zeros where there is none) is that after them
template <typename Acc> __global__ __launch_bounds__(GS_THREADS) void gscan_pass_kernel(const void *from, void *to, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * GS_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * GS_THREADS)
        static_cast<Acc *>(to)[i] = from == nullptr ? (Acc)0 : static_cast<const Acc *>(from)[i];
}
template <typename Acc> int pass(const void *from, void *to, int64_t n, hipStream_t stream) {
    if (to == nullptr) return T2FW_OK;
    const int64_t groups = (n + GS_THREADS - 1) / GS_THREADS;
    hipLaunchKernelGGL(gscan_pass_kernel<Acc>, dim3((unsigned)(groups < MOST_GROUPS ? groups : MOST_GROUPS)), dim3(GS_THREADS), 0, stream, from, to, n);
    return check_hip(hipGetLastError(), "gscan_pass_kernel launch");
}

// One token: x, f, out [B, D], the state in place or not.  A launch and a round to memory: 64 x 768 bf16 2.5 us.
template <typename IO, typename Acc, int VEC>
__global__ __launch_bounds__(GS_THREADS) void gscan_step_kernel(GscanArgs a, int64_t n) {
    const int64_t i = ((int64_t)blockIdx.x * GS_THREADS + threadIdx.x) * VEC;
    if (i >= n) return;
    const IO *x = static_cast<const IO *>(a.x), *f = static_cast<const IO *>(a.f);
    const Acc *s = static_cast<const Acc *>(a.s0);
    IO *out = static_cast<IO *>(a.out);
    Acc *next = static_cast<Acc *>(a.final_state);
    if (i + VEC <= n) {
        const Vec<IO, VEC> xv = load_vec<IO, VEC>(x + i), fv = load_vec<IO, VEC>(f + i);
        Vec<Acc, VEC> h = load_vec<Acc, VEC>(s + i);
        Vec<IO, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc z = widen(fv.e[v]);
            h.e[v] = (a.logits ? gate_of<IO>(z) : z) * h.e[v] + (Acc)widen(xv.e[v]);
            o.e[v] = narrow<IO>(h.e[v]);
        }
        store_vec(next + i, h);
        store_vec(out + i, o);
        return;
    }
    for (int64_t j = i; j < n; ++j) {
        const Acc z = widen(f[j]), h = (a.logits ? gate_of<IO>(z) : z) * s[j] + (Acc)widen(x[j]);
        next[j] = h;
        out[j] = narrow<IO>(h);
    }
}

// Channels of a workgroup: as few steps as fit, as long as there is a workgroup for every CU (4096 x 16 x 768 bf16 with logits, forward and
// backward: 303 and 497 us with 64 channels, 64 and 105 with 512; 8192 x 8 x 768: 546 and 932, 71 and 114 with 1024).
template <int VEC, int R> constexpr int64_t steps_of(int chn) { return GS_THREADS / (chn / VEC) * R; }
template <int VEC, int R> int channels_of(int64_t B, int64_t T, int64_t D) {
    const int64_t per_row = (D + VEC - 1) / VEC * VEC;
    for (int chn : {FEW_STEPS, 512, 256, 128})
        if (GS_THREADS >= chn / VEC && T <= steps_of<VEC, R>(chn) && B * per_row >= (int64_t)256 * chn) return chn;
    return GS_CHANNELS;
}
template <typename IO, int VEC, int R> GscanGrid grid_of(int64_t B, int64_t T, int64_t D) {
    GscanGrid g;
    g.channels = channels_of<VEC, R>(B, T, D);
    const int64_t CL = g.channels / VEC, C = steps_of<VEC, R>(g.channels);
    // (numbers that do not fit are refused before anything is launched)
    const int64_t per_row = (D + VEC - 1) / VEC, blocks = (B * per_row + CL - 1) / CL, chunks = T <= 0 ? 1 : (T + C - 1) / C;
    g.per_row = (uint32_t)per_row;
    g.blocks = (uint32_t)blocks;
    g.chunks = (uint32_t)chunks;
    g.fits = per_row < 0x7fffffff && B * per_row < 0x7fffffff && chunks <= MOST_GROUPS && blocks * chunks <= MOST_GROUPS;
    g.slots = blocks * g.channels;
    // With few workgroups the time is largely that of the wait: one group, so that nothing waits for a map made of maps (forward and backward
    // with the emptying launch: 1 x 8191 x 768 bf16, 768 workgroups, 18.3 and 22.0 us, in groups of 8 23.4 and 26.1; 2 x 8191 x 768, 1536 of
    // them, 24.7 and 33.1, 26.5 and 33.0; only 1 x 16384 x 768, 1536 of 128 chunks, loses by it: 28.7 and 36.8, in groups of 16 27.7 and
    // 34.5).  Otherwise the words read are what costs (1 x 16384 x 1024, 2048 workgroups: in groups of 16 30.1 and 46.1, one group 33.9 and 52.8;
    // 2 x 32768 x 1024 backward, 256 chunks: groups of 16 156, 32 161, 64 171, 128 185).  One or two workgroups side by side are between the
    // two, few words and long waits: groups twice as large (1 x 131072 x 128 bf16 forward and backward: 44 and 56 us, without 60 and 77;
    // of four workgroups side by side, 2 x 65536 x 128, the same either way).
    g.group = 8;
    if (chunks <= 128 && blocks * chunks < FEW_GROUPS) g.group = 128;
    while ((uint64_t)g.group * g.group < (uint64_t)chunks) g.group *= 2;
    if (blocks <= 2 && chunks > 128) g.group *= 2;
    return g;
}
// 64-bit words of the scratch
int64_t words_of(const GscanGrid &g) { return (g.chunks + (int64_t)(g.chunks + g.group - 1) / g.group) * g.slots; }

template <typename IO, int VEC, int R> GscanPlan plan_of(int64_t B, int64_t T, int64_t D) {
    const GscanGrid g = grid_of<IO, VEC, R>(B, T, D);
    const size_t acc = sizeof(typename AccT<IO>::type);
    GscanPlan p;
    p.checkpoints = (size_t)(g.chunks * g.slots) * acc;
    p.workspace = g.chunks == 1 ? 0 : acc == 8 ? (size_t)(g.chunks * g.slots) * 2 * acc : (size_t)words_of(g) * sizeof(uint64_t);
    return p;
}

// What comes before a call's main launch
template <typename IO, int VEC, int R, bool BACK, bool LOGITS> int prepare(const GscanArgs &a, const GscanGrid &g, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    if (!g.fits) return fail(T2FW_ERR_BAD_SHAPE, "gated scan: too many workgroups for one launch");
    if (g.chunks == 1) return T2FW_OK;
    if constexpr (sizeof(Acc) == 8) {
        hipLaunchKernelGGL((gscan_maps_kernel<IO, Acc, VEC, R, BACK, LOGITS>), dim3((unsigned)(g.blocks * (g.chunks - 1))), dim3(GS_THREADS), 0,
                           stream, a, g);
        return check_hip(hipGetLastError(), "gscan_maps_kernel launch");
    } else {
        const int64_t n = words_of(g);
        hipLaunchKernelGGL(gscan_empty_kernel, dim3((unsigned)((n + GS_THREADS - 1) / GS_THREADS)), dim3(GS_THREADS), 0, stream,
                           static_cast<uint64_t *>(a.words), n);
        return check_hip(hipGetLastError(), "gscan_empty_kernel launch");
    }
}

template <typename IO, int VEC, int R, bool LOGITS> int forward_with(const GscanArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    const GscanGrid g = grid_of<IO, VEC, R>(a.B, a.T, a.D);
    const int rc = prepare<IO, VEC, R, false, LOGITS>(a, g, stream);
    if (rc) return rc;
    const dim3 grid(g.blocks * g.chunks), threads(GS_THREADS);
    if (g.channels == GS_CHANNELS) hipLaunchKernelGGL((gscan_forward_kernel<IO, Acc, VEC, R, GS_CHANNELS, LOGITS>), grid, threads, 0, stream, a, g);
    if (g.channels == 128) hipLaunchKernelGGL((gscan_forward_kernel<IO, Acc, VEC, R, 128, LOGITS>), grid, threads, 0, stream, a, g);
    if constexpr (GS_THREADS >= 256 / VEC)
        if (g.channels == 256) hipLaunchKernelGGL((gscan_forward_kernel<IO, Acc, VEC, R, 256, LOGITS>), grid, threads, 0, stream, a, g);
    if constexpr (GS_THREADS >= 512 / VEC)
        if (g.channels == 512) hipLaunchKernelGGL((gscan_forward_kernel<IO, Acc, VEC, R, 512, LOGITS>), grid, threads, 0, stream, a, g);
    if constexpr (GS_THREADS >= FEW_STEPS / VEC)
        if (g.channels == FEW_STEPS) hipLaunchKernelGGL((gscan_forward_kernel<IO, Acc, VEC, R, FEW_STEPS, LOGITS>), grid, threads, 0, stream, a, g);
    return check_hip(hipGetLastError(), "gscan_forward_kernel launch");
}
template <typename IO, int VEC, int R> int forward_of(const GscanArgs &a, hipStream_t stream) {
    if (a.T == 0) return pass<typename AccT<IO>::type>(a.s0, a.final_state, a.B * a.D, stream);
    return a.logits ? forward_with<IO, VEC, R, true>(a, stream) : forward_with<IO, VEC, R, false>(a, stream);
}

template <typename IO, int VEC, int R, bool LOGITS> int backward_with(const GscanArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    const GscanGrid g = grid_of<IO, VEC, R>(a.B, a.T, a.D);
    const int rc = prepare<IO, VEC, R, true, LOGITS>(a, g, stream);
    if (rc) return rc;
    const dim3 grid(g.blocks * g.chunks), threads(GS_THREADS);
    if (g.channels == GS_CHANNELS) hipLaunchKernelGGL((gscan_backward_kernel<IO, Acc, VEC, R, GS_CHANNELS, LOGITS>), grid, threads, 0, stream, a, g);
    if (g.channels == 128) hipLaunchKernelGGL((gscan_backward_kernel<IO, Acc, VEC, R, 128, LOGITS>), grid, threads, 0, stream, a, g);
    if constexpr (GS_THREADS >= 256 / VEC)
        if (g.channels == 256) hipLaunchKernelGGL((gscan_backward_kernel<IO, Acc, VEC, R, 256, LOGITS>), grid, threads, 0, stream, a, g);
    if constexpr (GS_THREADS >= 512 / VEC)
        if (g.channels == 512) hipLaunchKernelGGL((gscan_backward_kernel<IO, Acc, VEC, R, 512, LOGITS>), grid, threads, 0, stream, a, g);
    if constexpr (GS_THREADS >= FEW_STEPS / VEC)
        if (g.channels == FEW_STEPS) hipLaunchKernelGGL((gscan_backward_kernel<IO, Acc, VEC, R, FEW_STEPS, LOGITS>), grid, threads, 0, stream, a, g);
    return check_hip(hipGetLastError(), "gscan_backward_kernel launch");
}
template <typename IO, int VEC, int R> int backward_of(const GscanArgs &a, hipStream_t stream) {
    if (a.T == 0) return pass<typename AccT<IO>::type>(a.g_state, a.d_s0, a.B * a.D, stream);
    return a.logits ? backward_with<IO, VEC, R, true>(a, stream) : backward_with<IO, VEC, R, false>(a, stream);
}

template <typename IO> int step_of(const GscanArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    constexpr int VEC = 16 / sizeof(IO);
    const int64_t n = a.B * a.D, groups = (n + (int64_t)GS_THREADS * VEC - 1) / ((int64_t)GS_THREADS * VEC);
    if (groups > MOST_GROUPS) return fail(T2FW_ERR_BAD_SHAPE, "gated scan: too many channels for one launch");
    hipLaunchKernelGGL((gscan_step_kernel<IO, Acc, VEC>), dim3((unsigned)groups), dim3(GS_THREADS), 0, stream, a, n);
    return check_hip(hipGetLastError(), "gscan_step_kernel launch");
}

// rows narrower than a lane's vector go channel by channel
#define GSCAN_OF(IO, what, ...) (a.D >= Tile<IO>::VEC ? what<IO, Tile<IO>::VEC, Tile<IO>::R>(__VA_ARGS__) : what<IO, 1, 8>(__VA_ARGS__))

}  // namespace

GscanPlan gscan_plan(int64_t B, int64_t T, int64_t D, int dtype) {
    struct { int64_t D; } a{D};
    switch (dtype) {
        case T2FW_F32: return GSCAN_OF(float, plan_of, B, T, D);
        case T2FW_F64: return GSCAN_OF(double, plan_of, B, T, D);
    }
    return GSCAN_OF(_Float16, plan_of, B, T, D);
}

int gscan_forward(const GscanArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return GSCAN_OF(float, forward_of, a, stream);
        case T2FW_F16: return GSCAN_OF(_Float16, forward_of, a, stream);
        case T2FW_BF16: return GSCAN_OF(__bf16, forward_of, a, stream);
    }
    return GSCAN_OF(double, forward_of, a, stream);
}

int gscan_backward(const GscanArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return GSCAN_OF(float, backward_of, a, stream);
        case T2FW_F16: return GSCAN_OF(_Float16, backward_of, a, stream);
        case T2FW_BF16: return GSCAN_OF(__bf16, backward_of, a, stream);
    }
    return GSCAN_OF(double, backward_of, a, stream);
}

int gscan_step(const GscanArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return step_of<float>(a, stream);
        case T2FW_F16: return step_of<_Float16>(a, stream);
        case T2FW_BF16: return step_of<__bf16>(a, stream);
    }
    return step_of<double>(a, stream);
}

}  // namespace t2fw
