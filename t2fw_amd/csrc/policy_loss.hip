// The clipped policy loss with a KL term, from the logits of the tokens, and its gradient.  For a token with logits z, target t,
//   logp = z_t - lse(z),  r = exp(logp - old),  d = ref - logp,
//   loss = scale / M  sum over the M tokens of the mask of  -min(r A, clip(r, low, high) A) + kl (exp(d) - 1 - d)
//   d loss / d z = c (onehot(t) - softmax(z)),  c = scale / M (-r A [not held by the clip] - kl (exp(d) - 1)).
// The coefficient c of a row depends on nothing but the row and M, so that the launch that reads a row for its log-sum-exp
// writes its gradient too, for a gradient of the loss of one; the backward has nothing left to do then but to look at that value.
// The log-sum-exp is never one number: with m the largest logit and s = sum exp(z - m), logp = (z_t - m) - log s and softmax = exp(z - m) / s,
// so that logits with a common offset lose nothing to it.
//
// Bound by memory: 8192 x 50257 bf16, loss and gradient, 315 us (1.65 GB of logits and gradient, 5.2 TB/s, as a copy); with the gradient in a pass
// of its own the logits would be read twice.  Few rows are bound by the chain load, exchange, exponentials, store: 333 x 8000
// float32 13.5 us, 4 for the sum of the tokens' shares and 2 for the backward's look.
#include "policy_loss.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

// 16-bit logits: the hardware's exponential, off by |v| 1.25 2^-24 (the argument is rounded to 32 bits once multiplied by log2 e) and 2^-22: 2^-19
// at a logit 20 below the largest, whose term is 2^-29 of the largest's; the logits' own rounding is worth 2^-12 or 2^-9 of them.  32-bit ones: the library's, with
// which 8192 x 50257 bf16 would take 493 us for 325.
template <typename IO> __device__ __forceinline__ float exp_of(float v) { return sizeof(IO) == 2 ? __expf(v) : expf(v); }

constexpr int PL_THREADS = 1024;

// A maximum and a sum of exponentials over it; what minus infinity stands for is nothing
struct Top {
    float m, s;
};
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
template <typename IO> __device__ __forceinline__ Top joined(const Top &a, const Top &b) {
    // two products and a sum, not a fused form: the lanes of a pair, which see a and b the other way round, get the same bits
#pragma clang fp contract(off)
    const float m = fmaxf(a.m, b.m), base = base_of(m);
    return {m, a.s * exp_of<IO>(a.m - base) + b.s * exp_of<IO>(b.m - base)};
}
template <typename IO> __device__ __forceinline__ Top joined_lanes(Top t, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) t = joined<IO>(t, {__shfl_xor(t.m, m, 64), __shfl_xor(t.s, m, 64)});
    return t;
}

struct TokenTerms {
    float loss, coef;
};
// one token's share of the loss and its row's coefficient, both without scale / M
__device__ __forceinline__ TokenTerms terms_of(const PolicyLossArgs &a, int64_t row, float logp) {
    const float adv = a.adv[row], r = expf(logp - a.old_logp[row]);
    const float freely = r * adv, held = fminf(fmaxf(r, a.low), a.high) * adv;
    const bool moves = freely < held || (r >= a.low && r <= a.high) || r != r;
    // the clip's comparisons drop a NaN that the sums keep
    const TokenTerms clipped{r != r ? r : -fminf(freely, held), moves ? -freely : 0.0f};
    // left out rather than multiplied by zero: without a reference its log probabilities are anything, and exp(ref - logp) may be infinite
    if (a.kl == 0.0f) return clipped;
    const float d = a.ref_logp[row] - logp, em = expm1f(d);
    return {clipped.loss + a.kl * (em - d), clipped.coef - a.kl * em};
}

// What a workgroup needs besides a row: the number of tokens that count.  Every workgroup counts them itself as long as that is 16 bytes
// for each thread; a launch of its own does it for more.
constexpr int64_t COUNTED_BYTES = 16;
template <int THREADS> __device__ __forceinline__ int64_t counted(const PolicyLossArgs &a) {
    __shared__ int64_t parts[THREADS / 64];
    int64_t n = 0;
    for (int64_t i = (int64_t)threadIdx.x * 8; i < a.N; i += THREADS * 8) {
        if (i + 8 <= a.N) {
            const Vec<uint8_t, 8> v = load_vec<uint8_t, 8>(a.mask + i);
#pragma unroll
            for (int j = 0; j < 8; ++j) n += v.e[j] != 0;
        } else {
            for (int64_t j = i; j < a.N; ++j) n += a.mask[j] != 0;
        }
    }
    for (int m = 1; m < 64; m <<= 1) n += __shfl_xor(n, m, 64);
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = n;
    __syncthreads();
    n = 0;
    for (int i = 0; i < THREADS / 64; ++i) n += parts[i];
    return n;
}
__global__ __launch_bounds__(PL_THREADS) void policy_count_kernel(PolicyLossArgs a) {
    const int64_t n = counted<PL_THREADS>(a);
    if (threadIdx.x == 0) *a.tokens = n;
}

// A row in the registers of a workgroup: CH vectors of each thread.  Rows of an odd vocabulary start anywhere, and loads and
// stores that are not aligned cost a fifth of the rate (8192 x 50257 bfloat16: 388 us, 325 for 50264): the vectors begin at the first aligned
// element, and the few before them and after the last whole one are one each for the first threads.
template <typename IO, int THREADS, int CH> struct Row {
    static constexpr int VEC = 16 / sizeof(IO);
    Raw16 v[CH];
    float extra;                        // minus infinity where there is none
    int head, vectors, rest;            // elements before the vectors, the vectors, elements after them
    __device__ __forceinline__ static int at(int c) { return c * THREADS + (int)threadIdx.x; }
    __device__ __forceinline__ int extra_at() const { return (int)threadIdx.x < head ? (int)threadIdx.x : head + vectors * VEC + (int)threadIdx.x - head; }
    __device__ __forceinline__ bool has_extra() const { return (int)threadIdx.x < head + rest; }
    __device__ __forceinline__ void load(const IO *z, int64_t V) {
        const int to_aligned = (int)((16 - reinterpret_cast<uintptr_t>(z) % 16) % 16 / sizeof(IO));
        head = to_aligned < V ? to_aligned : (int)V;
        vectors = ((int)V - head) / VEC;
        rest = (int)V - head - vectors * VEC;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (at(c) < vectors) v[c] = load_raw(z + head + (int64_t)at(c) * VEC);
        extra = has_extra() ? (float)widen(z[extra_at()]) : -INFINITY;
    }
    // The row is held as it came: without this the compiler keeps its 32-bit form from one use to the next, in twice the registers
    __device__ __forceinline__ void stay_narrow() {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(v[c].w[i]));
    }
    __device__ __forceinline__ Top top(int64_t) {
        float m = extra;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (at(c) < vectors) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) m = fmaxf(m, element<IO>(v[c], j));
            }
        const float base = base_of(m);
        float s = exp_of<IO>(extra - base);
        stay_narrow();
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (at(c) < vectors) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) s += exp_of<IO>(element<IO>(v[c], j) - base);
            }
        stay_narrow();
        return {m, s};
    }
    // -c softmax = -per exp(z - base), and at the target, by the thread that has just written there, c more
    __device__ __forceinline__ void gradient(IO *dz, int64_t V, float base, float per, float c, int64_t target, float logp) const {
#pragma unroll
        for (int k = 0; k < CH; ++k)
            if (at(k) < vectors) {
                Vec<IO, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) o.e[j] = narrow<IO>(-per * exp_of<IO>(element<IO>(v[k], j) - base));
                store_vec(dz + head + (int64_t)at(k) * VEC, o);
            }
        if (has_extra()) dz[extra_at()] = narrow<IO>(-per * exp_of<IO>(extra - base));
        if (target >= 0 && target < V) {
            const int t = (int)target, in = t - head;
            const int owner = t < head ? t : in < vectors * VEC ? in / VEC % THREADS : head + in - vectors * VEC;
            if ((int)threadIdx.x == owner) dz[t] = narrow<IO>(fmaf(-c, exp_of<IO>(logp), c));
        }
    }
    __device__ __forceinline__ void zeros(IO *dz, int64_t) const {
#pragma unroll
        for (int k = 0; k < CH; ++k)
            if (at(k) < vectors) store_vec(dz + head + (int64_t)at(k) * VEC, Vec<IO, VEC>{});
        if (has_extra()) dz[extra_at()] = (IO)0;
    }
};

// The same for a row that does not fit: read twice, the second time from a cache
template <typename IO, int THREADS> struct Row<IO, THREADS, 0> {
    static constexpr int VEC = 16 / sizeof(IO);
    const IO *z;
    __device__ __forceinline__ void load(const IO *row, int64_t) { z = row; }
    __device__ __forceinline__ Top top(int64_t V) const {
        Top t{-INFINITY, 0};
        for (int64_t i = (int64_t)threadIdx.x * VEC; i < V; i += THREADS * VEC) {
            float v[VEC], m = t.m;
            if (i + VEC <= V) {
                const Vec<IO, VEC> raw = load_vec<IO, VEC>(z + i);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = widen(raw.e[j]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = i + j < V ? (float)widen(z[i + j]) : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) m = fmaxf(m, v[j]);
            const float base = base_of(m);
            t.s *= exp_of<IO>(t.m - base);
            t.m = m;
#pragma unroll
            for (int j = 0; j < VEC; ++j) t.s += exp_of<IO>(v[j] - base);
        }
        return t;
    }
    __device__ __forceinline__ void gradient(IO *dz, int64_t V, float base, float per, float c, int64_t target, float logp) const {
        for (int64_t i = (int64_t)threadIdx.x * VEC; i < V; i += THREADS * VEC) {
            if (i + VEC <= V) {
                const Vec<IO, VEC> v = load_vec<IO, VEC>(z + i);
                Vec<IO, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) o.e[j] = narrow<IO>(-per * exp_of<IO>(widen(v.e[j]) - base));
                store_vec(dz + i, o);
            } else {
                for (int64_t j = i; j < V; ++j) dz[j] = narrow<IO>(-per * exp_of<IO>(widen(z[j]) - base));
            }
            if (target >= i && target < i + VEC && target < V) dz[target] = narrow<IO>(fmaf(-c, exp_of<IO>(logp), c));
        }
    }
    __device__ __forceinline__ void zeros(IO *dz, int64_t V) const {
        for (int64_t i = (int64_t)threadIdx.x * VEC; i < V; i += THREADS * VEC) {
            if (i + VEC <= V) store_vec(dz + i, Vec<IO, VEC>{});
            else
                for (int64_t j = i; j < V; ++j) dz[j] = (IO)0;
        }
    }
};

// GROUPS workgroups share a CU: what a row's loads and stores leave idle is another's
template <typename IO, int THREADS, int CH, int GROUPS>
__global__ __launch_bounds__(THREADS, GROUPS * THREADS / 256) void policy_rows_kernel(PolicyLossArgs a) {
    constexpr int WAVES = THREADS / 64;
    __shared__ Top tops[2][WAVES];
    const int64_t M = a.mask == nullptr ? a.N : a.N > COUNTED_BYTES * THREADS ? *a.tokens : counted<THREADS>(a);
    const float share = a.scale / (float)(M > 0 ? M : 1);
    double sum = 0;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x, turn ^= 1) {
        const IO *z = static_cast<const IO *>(a.logits) + row * a.V;
        const int64_t t = a.targets[row];
        const bool counts = a.mask == nullptr || a.mask[row] != 0, known = t >= 0 && t < a.V;
        const float zt = known ? (float)widen(z[t]) : 0.0f;
        Row<IO, THREADS, CH> r;
        r.load(z, a.V);
        Top top = joined_lanes<IO>(r.top(a.V), 64);
        if (threadIdx.x % 64 == 0) tops[turn][threadIdx.x / 64] = top;
        __syncthreads();                                 // (the other half is free again: every wave has read it before this row's barrier)
        top = joined_lanes<IO>(tops[turn][threadIdx.x % WAVES], WAVES);
        const float base = base_of(top.m), logp = known ? zt - base - logf(top.s) : counts ? NAN : 0.0f;
        TokenTerms m{0, 0};
        if (counts) m = terms_of(a, row, logp);
        if (threadIdx.x == 0) {
            a.logp[row] = logp;
            a.tops[2 * row] = base;
            a.tops[2 * row + 1] = top.s;
            a.coef[row] = m.coef * share;
            sum += (double)(m.loss * share);
        }
        if (a.d_logits != nullptr) {
            IO *const dz = static_cast<IO *>(a.d_logits) + row * a.V;
            if (counts) r.gradient(dz, a.V, base, m.coef * share / top.s, m.coef * share, t, logp);
            else r.zeros(dz, a.V);
        }
    }
    if (threadIdx.x == 0) a.sums[blockIdx.x] = sum;
}

// The loss: the workgroups' sums, in order
constexpr int PS_THREADS = 1024;
__global__ __launch_bounds__(PS_THREADS) void policy_sum_kernel(const double *sums, int n, float *loss) {
    __shared__ double parts[PS_THREADS / 64];
    double s = 0;
    for (int i = threadIdx.x; i < n; i += PS_THREADS) s += sums[i];
    s = group_sum(s, 64);
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < PS_THREADS / 64; ++i) s += parts[i];
        *loss = (float)s;
    }
}

template <typename IO>
__global__ __launch_bounds__(PL_THREADS) void policy_gradient_kernel(PolicyLossArgs a) {
    const float g = *a.g_loss;
    if (a.unless_one && g == 1.0f) return;
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
        const IO *z = static_cast<const IO *>(a.logits) + row * a.V;
        IO *const dz = static_cast<IO *>(a.d_logits) + row * a.V;
        const int64_t t = a.targets[row];
        const float base = a.tops[2 * row], s = a.tops[2 * row + 1], c = a.coef[row] * g;
        const float logp = t >= 0 && t < a.V ? widen(z[t]) - base - logf(s) : 0.0f;
        Row<IO, PL_THREADS, 0> r;
        r.load(z, a.V);
        if (c == 0.0f) r.zeros(dz, a.V);
        else r.gradient(dz, a.V, base, c / s, c, t, logp);
    }
}

// Workgroups of a launch over all rows: as many as the chip holds
int groups_of(int64_t N, int64_t resident) { return (int)(N < resident ? N : resident); }

template <typename IO> int forward_of(const PolicyLossArgs &a, hipStream_t stream) {
    constexpr int VEC = 16 / sizeof(IO);
    int groups = 0;
#define POLICY_ROWS(THREADS, CH, GROUPS)                                                                                            \
    do {                                                                                                                            \
        groups = groups_of(a.N, 256 * GROUPS);                                                                                      \
        if (a.mask != nullptr && a.N > COUNTED_BYTES * THREADS)                                                                     \
            hipLaunchKernelGGL(policy_count_kernel, dim3(1), dim3(PL_THREADS), 0, stream, a);                                       \
        hipLaunchKernelGGL((policy_rows_kernel<IO, THREADS, CH, GROUPS>), dim3((unsigned)groups), dim3(THREADS), 0, stream, a);     \
    } while (0)
    if (a.N > 0) {
        const int64_t vectors = a.V / VEC;
        // A short row leaves most of a large workgroup idle in its exchange, a long one needs the registers of many threads; in between,
        // several rows on a CU hide each other's loads and stores.  bfloat16, TB/s of logits and gradient (a copy of this size: 5.2):
        //   16384 x 1000   one wave 2.10, 256 threads 1.49             16384 x 3500   one wave 3.60, 256 threads 3.41, 1024 threads 2
        //   16384 x 12001  256 threads 4.62, 512 4.13, 1024 3.21       8192 x 32000   2 x 512 threads 5.09, 1024 threads 4.59
        //   8192 x 50257   1024 threads 5.23, 2 x 512 4.95, 2 x 1024 (64 registers) 4.59, row read twice 3.26
        if (vectors <= 2 * 64) POLICY_ROWS(64, 2, 32);
        else if (vectors <= 7 * 64) POLICY_ROWS(64, 7, 16);
        else if (vectors <= 4 * 256) POLICY_ROWS(256, 4, 8);
        else if (vectors <= 7 * 256) POLICY_ROWS(256, 7, 6);
        else if (vectors <= 8 * 512) POLICY_ROWS(512, 8, 3);
        else if (vectors <= 11 * 512) POLICY_ROWS(512, 11, 2);
        else if (vectors <= 8 * 1024) POLICY_ROWS(1024, 8, 1);
        else if (vectors <= 16 * 1024) POLICY_ROWS(1024, 16, 1);
        else POLICY_ROWS(1024, 0, 2);
        const int rc = check_hip(hipGetLastError(), "policy_rows_kernel launch");
        if (rc) return rc;
    }
#undef POLICY_ROWS
    hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(PS_THREADS), 0, stream, a.sums, groups, a.loss);
    return check_hip(hipGetLastError(), "policy_sum_kernel launch");
}

template <typename IO> int backward_of(const PolicyLossArgs &a, hipStream_t stream) {
    if (a.N == 0) return T2FW_OK;
    hipLaunchKernelGGL(policy_gradient_kernel<IO>, dim3((unsigned)groups_of(a.N, 512)), dim3(PL_THREADS), 0, stream, a);
    return check_hip(hipGetLastError(), "policy_gradient_kernel launch");
}

}  // namespace

int policy_loss_forward(const PolicyLossArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return forward_of<float>(a, stream);
        case T2FW_F16: return forward_of<_Float16>(a, stream);
    }
    return forward_of<__bf16>(a, stream);
}

int policy_loss_backward(const PolicyLossArgs &a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case T2FW_F32: return backward_of<float>(a, stream);
        case T2FW_F16: return backward_of<_Float16>(a, stream);
    }
    return backward_of<__bf16>(a, stream);
}

}  // namespace t2fw
