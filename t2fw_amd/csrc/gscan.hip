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
#include "gscan.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int GS_THREADS = 256;
constexpr int GS_CHANNELS = 64;          // channels of a workgroup

// elements of a lane: 32 in all, whatever the type
template <typename IO> struct Tile {
    static constexpr int VEC = 16 / sizeof(IO), R = 32 / VEC;
};
template <typename IO> struct AccT { using type = float; };
template <> struct AccT<double> { using type = double; };

template <typename Acc> struct Map {
    Acc p, s;
};

template <typename IO> __device__ __forceinline__ float gate_of(float z) {
    // 16-bit gates: hardware exponential and reciprocal (2^-21); 32-bit ones: the library's
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
template <int VEC, int R>
__device__ __forceinline__ Place<VEC, R> place_of(const GscanArgs &a, int64_t per_row, int64_t block, int64_t chunk) {
    constexpr int CL = GS_CHANNELS / VEC, TG = GS_THREADS / CL;
    Place<VEC, R> p;
    p.lane = threadIdx.x % CL;
    p.group = threadIdx.x / CL;
    p.slot = block * CL + p.lane;
    p.mine = p.slot < a.B * per_row;
    p.b = p.mine ? p.slot / per_row : 0;
    const int64_t d = (p.slot - p.b * per_row) * VEC;
    p.d = d + VEC <= a.D ? d : a.D - VEC;
    p.t0 = chunk * (TG * R) + (int64_t)p.group * R;
    const int64_t left = p.mine ? a.T - p.t0 : 0, live = p.mine ? row_length(a, p.b) - p.t0 : 0;
    p.steps = left < 0 ? 0 : left < R ? (int)left : R;
    p.live = live < 0 ? 0 : live < R ? (int)live : R;
    return p;
}

template <typename IO, int VEC, int R>
__device__ __forceinline__ void load_steps(Vec<IO, VEC> (&v)[R], const void *base, int64_t row, int64_t step, const Place<VEC, R> &p) {
    const IO *at = static_cast<const IO *>(base) + p.b * row + p.t0 * step + p.d;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r < p.live) v[r] = load_vec<IO, VEC>(at + r * step);
}

// What a step beyond the row's length holds does not count, whatever it is: gate one, input nothing
template <typename IO, typename Acc, int VEC, int R>
__device__ __forceinline__ void gates_of(Acc (&g)[R][VEC], const Vec<IO, VEC> (&f)[R], const Place<VEC, R> &p, int logits) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Acc z = widen(f[r].e[v]);
            g[r][v] = r < p.live ? (logits ? gate_of<IO>(z) : z) : (Acc)1;
        }
}
template <typename IO, typename Acc, int VEC, int R>
__device__ __forceinline__ Acc value_of(const Vec<IO, VEC> (&x)[R], int r, int v, const Place<VEC, R> &p) {
    return r < p.live ? (Acc)widen(x[r].e[v]) : (Acc)0;
}

// The map of every channel over a stretch, forward in time, or of its adjoint, backward
template <typename IO, typename Acc, int VEC, int R, bool BACK>
__device__ __forceinline__ void fold_steps(Map<Acc> (&m)[VEC], const Acc (&g)[R][VEC], const Vec<IO, VEC> (&x)[R], const Place<VEC, R> &p) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Acc pr = 1, s = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = BACK ? R - 1 - i : i;
            const Acc in = value_of<IO, Acc, VEC, R>(x, r, v, p);
            s = BACK ? g[r][v] * (s + in) : g[r][v] * s + in;
            pr *= g[r][v];
        }
        m[v].p = pr;
        m[v].s = s;
    }
}

// The map of a whole chunk, for what comes after it in the direction of the recurrence
template <typename IO, typename Acc, int VEC, int R, bool BACK>
__global__ __launch_bounds__(GS_THREADS) void gscan_maps_kernel(GscanArgs a, int64_t per_row, int64_t blocks, int64_t slots) {
    constexpr int CL = GS_CHANNELS / VEC, TG = GS_THREADS / CL;
    __shared__ Map<Acc> maps[TG][GS_CHANNELS];
    const int64_t block = blockIdx.x % blocks, chunk = blockIdx.x / blocks + (BACK ? 1 : 0);
    const Place<VEC, R> p = place_of<VEC, R>(a, per_row, block, chunk);
    Vec<IO, VEC> x[R], f[R];
    load_steps(f, a.f, a.f_b, a.f_t, p);
    load_steps(x, BACK ? a.g_out : a.x, BACK ? a.g_b : a.x_b, BACK ? a.g_t : a.x_t, p);
    Acc g[R][VEC];
    gates_of<IO, Acc, VEC, R>(g, f, p, a.logits);
    Map<Acc> m[VEC];
    fold_steps<IO, Acc, VEC, R, BACK>(m, g, x, p);
#pragma unroll
    for (int v = 0; v < VEC; ++v) maps[p.group][p.lane * VEC + v] = m[v];
    __syncthreads();
    if (threadIdx.x >= GS_CHANNELS) return;
    Acc pr = 1, s = 0;
#pragma unroll
    for (int i = 0; i < TG; ++i) {
        const Map<Acc> m2 = maps[BACK ? TG - 1 - i : i][threadIdx.x];
        s = m2.p * s + m2.s;
        pr *= m2.p;
    }
    static_cast<Map<Acc> *>(a.words)[chunk * slots + block * GS_CHANNELS + threadIdx.x] = Map<Acc>{pr, s};
}

// The channel of a workgroup's thread in [B, D] arrays; whether it is there
template <int VEC> __device__ __forceinline__ bool channel_of(const GscanArgs &a, int64_t per_row, int64_t block, int64_t *at) {
    const int64_t slot = block * (GS_CHANNELS / VEC) + threadIdx.x / VEC, b = slot / per_row, d = (slot - b * per_row) * VEC;
    *at = b * a.D + (d + VEC <= a.D ? d : a.D - VEC) + threadIdx.x % VEC;
    return slot < a.B * per_row;
}

template <typename IO, typename Acc, int VEC, int R>
__global__ __launch_bounds__(GS_THREADS) void gscan_forward_kernel(GscanArgs a, int64_t per_row, int64_t blocks, int64_t chunks, int64_t slots) {
    constexpr int CL = GS_CHANNELS / VEC, TG = GS_THREADS / CL;
    __shared__ Map<Acc> maps[TG][GS_CHANNELS];
    const int64_t block = blockIdx.x % blocks, chunk = blockIdx.x / blocks;
    const Place<VEC, R> p = place_of<VEC, R>(a, per_row, block, chunk);
    Vec<IO, VEC> x[R], f[R];
    load_steps(f, a.f, a.f_b, a.f_t, p);
    load_steps(x, a.x, a.x_b, a.x_t, p);
    Acc g[R][VEC];
    gates_of<IO, Acc, VEC, R>(g, f, p, a.logits);
    {
        Map<Acc> m[VEC];
        fold_steps<IO, Acc, VEC, R, false>(m, g, x, p);
#pragma unroll
        for (int v = 0; v < VEC; ++v) maps[p.group][p.lane * VEC + v] = m[v];
    }
    __syncthreads();
    if (threadIdx.x < GS_CHANNELS) {
        int64_t at;
        const bool there = channel_of<VEC>(a, per_row, block, &at);
        Acc h = there && a.s0 != nullptr ? static_cast<const Acc *>(a.s0)[at] : (Acc)0;
        const int64_t column = block * GS_CHANNELS + threadIdx.x;
        const Map<Acc> *w = static_cast<const Map<Acc> *>(a.words) + column;
        for (int64_t c = 0; c < chunk; ++c) h = w[c * slots].p * h + w[c * slots].s;
        if (a.ckpt != nullptr) static_cast<Acc *>(a.ckpt)[chunk * slots + column] = h;
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            const Map<Acc> m2 = maps[i][threadIdx.x];
            maps[i][threadIdx.x].s = h;                  // the state before this stretch
            h = m2.p * h + m2.s;
        }
        if (there && chunk == chunks - 1) static_cast<Acc *>(a.final_state)[at] = h;
    }
    __syncthreads();
    Vec<IO, VEC> o[R];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Acc h = maps[p.group][p.lane * VEC + v].s;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            h = g[r][v] * h + value_of<IO, Acc, VEC, R>(x, r, v, p);
            o[r].e[v] = r < p.live ? narrow<IO>(h) : narrow<IO>((Acc)0);
        }
    }
    IO *at = static_cast<IO *>(a.out) + (p.b * a.T + p.t0) * a.D + p.d;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r < p.steps) store_vec(at + r * a.D, o[r]);
}

template <typename IO, typename Acc, int VEC, int R>
__global__ __launch_bounds__(GS_THREADS) void gscan_backward_kernel(GscanArgs a, int64_t per_row, int64_t blocks, int64_t chunks, int64_t slots) {
    constexpr int CL = GS_CHANNELS / VEC, TG = GS_THREADS / CL;
    __shared__ Map<Acc> maps[TG][GS_CHANNELS];           // states: forward in time
    __shared__ Acc sums[TG][GS_CHANNELS];                // adjoints: backward, with the same gate products
    const int64_t block = blockIdx.x % blocks, chunk = chunks - 1 - blockIdx.x / blocks;
    const Place<VEC, R> p = place_of<VEC, R>(a, per_row, block, chunk);
    Vec<IO, VEC> x[R], f[R], go[R];
    load_steps(f, a.f, a.f_b, a.f_t, p);
    load_steps(go, a.g_out, a.g_b, a.g_t, p);
    load_steps(x, a.x, a.x_b, a.x_t, p);
    Acc g[R][VEC];
    gates_of<IO, Acc, VEC, R>(g, f, p, a.logits);
    {
        Map<Acc> m[VEC], n[VEC];
        fold_steps<IO, Acc, VEC, R, true>(n, g, go, p);
        fold_steps<IO, Acc, VEC, R, false>(m, g, x, p);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            maps[p.group][p.lane * VEC + v] = m[v];
            sums[p.group][p.lane * VEC + v] = n[v].s;
        }
    }
    __syncthreads();
    if (threadIdx.x < GS_CHANNELS) {
        int64_t at;
        const bool there = channel_of<VEC>(a, per_row, block, &at);
        const int64_t column = block * GS_CHANNELS + threadIdx.x;
        Acc e = there && a.g_state != nullptr ? static_cast<const Acc *>(a.g_state)[at] : (Acc)0;
        const Map<Acc> *w = static_cast<const Map<Acc> *>(a.words) + column;
        for (int64_t c = chunks - 1; c > chunk; --c) e = w[c * slots].p * e + w[c * slots].s;
        Acc h = static_cast<const Acc *>(a.ckpt)[chunk * slots + column];
        Acc pr[TG];
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            const Map<Acc> m2 = maps[i][threadIdx.x];
            maps[i][threadIdx.x].s = h;
            pr[i] = m2.p;
            h = m2.p * h + m2.s;
        }
#pragma unroll
        for (int i = TG - 1; i >= 0; --i) {
            const Acc s = sums[i][threadIdx.x];
            sums[i][threadIdx.x] = e;                    // the adjoint after this stretch
            e = pr[i] * e + s;
        }
        if (there && chunk == 0 && a.d_s0 != nullptr) static_cast<Acc *>(a.d_s0)[at] = e;
    }
    __syncthreads();
    Vec<IO, VEC> dx[R], df[R];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        Acc h = maps[p.group][p.lane * VEC + v].s, before[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            before[r] = h;
            h = g[r][v] * h + value_of<IO, Acc, VEC, R>(x, r, v, p);
        }
        Acc e = sums[p.group][p.lane * VEC + v];
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            const Acc d = value_of<IO, Acc, VEC, R>(go, r, v, p) + e;
            e = g[r][v] * d;
            Acc slope = d * before[r];
            if (a.logits) slope *= gate_slope<IO>((Acc)widen(f[r].e[v]));
            dx[r].e[v] = narrow<IO>(r < p.live ? d : (Acc)0);
            df[r].e[v] = narrow<IO>(r < p.live ? slope : (Acc)0);
        }
    }
    const int64_t at = (p.b * a.T + p.t0) * a.D + p.d;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r < p.steps) {
            store_vec(static_cast<IO *>(a.d_x) + at + r * a.D, dx[r]);
            store_vec(static_cast<IO *>(a.d_f) + at + r * a.D, df[r]);
        }
}

// One token: x, f, out [B, D], the state in place or not
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

template <typename IO, int VEC, int R> int64_t slots_per_row(int64_t D) { return (D + VEC - 1) / VEC; }

template <typename IO, int VEC, int R> GscanPlan plan_of(int64_t B, int64_t T, int64_t D) {
    constexpr int CL = GS_CHANNELS / VEC, TG = GS_THREADS / CL;
    GscanPlan p;
    p.chunk = TG * R;
    p.chunks = T <= 0 ? 1 : (T + p.chunk - 1) / p.chunk;
    p.slots = (B * slots_per_row<IO, VEC, R>(D) + CL - 1) / CL * GS_CHANNELS;
    p.acc = sizeof(typename AccT<IO>::type);
    return p;
}

int too_large() { return fail(T2FW_ERR_BAD_SHAPE, "gated scan: too many workgroups for one launch"); }

template <typename IO, int VEC, int R> int forward_of(const GscanArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    const GscanPlan p = plan_of<IO, VEC, R>(a.B, a.T, a.D);
    const int64_t per_row = slots_per_row<IO, VEC, R>(a.D), blocks = p.slots / GS_CHANNELS;
    if (blocks > 0x7fffffff / p.chunks) return too_large();
    if (p.chunks > 1) {
        hipLaunchKernelGGL((gscan_maps_kernel<IO, Acc, VEC, R, false>), dim3((unsigned)(blocks * (p.chunks - 1))), dim3(GS_THREADS), 0, stream, a,
                           per_row, blocks, p.slots);
        const int rc = check_hip(hipGetLastError(), "gscan_maps_kernel launch");
        if (rc) return rc;
    }
    hipLaunchKernelGGL((gscan_forward_kernel<IO, Acc, VEC, R>), dim3((unsigned)(blocks * p.chunks)), dim3(GS_THREADS), 0, stream, a, per_row,
                       blocks, p.chunks, p.slots);
    return check_hip(hipGetLastError(), "gscan_forward_kernel launch");
}

template <typename IO, int VEC, int R> int backward_of(const GscanArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    const GscanPlan p = plan_of<IO, VEC, R>(a.B, a.T, a.D);
    const int64_t per_row = slots_per_row<IO, VEC, R>(a.D), blocks = p.slots / GS_CHANNELS;
    if (blocks > 0x7fffffff / p.chunks) return too_large();
    if (p.chunks > 1) {
        hipLaunchKernelGGL((gscan_maps_kernel<IO, Acc, VEC, R, true>), dim3((unsigned)(blocks * (p.chunks - 1))), dim3(GS_THREADS), 0, stream, a,
                           per_row, blocks, p.slots);
        const int rc = check_hip(hipGetLastError(), "gscan_maps_kernel launch");
        if (rc) return rc;
    }
    hipLaunchKernelGGL((gscan_backward_kernel<IO, Acc, VEC, R>), dim3((unsigned)(blocks * p.chunks)), dim3(GS_THREADS), 0, stream, a, per_row,
                       blocks, p.chunks, p.slots);
    return check_hip(hipGetLastError(), "gscan_backward_kernel launch");
}

template <typename IO> int step_of(const GscanArgs &a, hipStream_t stream) {
    using Acc = typename AccT<IO>::type;
    constexpr int VEC = 16 / sizeof(IO);
    const int64_t n = a.B * a.D, groups = (n + (int64_t)GS_THREADS * VEC - 1) / ((int64_t)GS_THREADS * VEC);
    if (groups > 0x7fffffff) return too_large();
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
