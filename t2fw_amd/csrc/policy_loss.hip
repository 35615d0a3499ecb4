// The clipped policy loss with a KL term, from the logits of the tokens, and its gradient.  For a token with logits z, target t,
//   logp = z_t - lse(z),  r = exp(logp - old),  d = ref - logp,
//   loss = scale / M  sum over the M tokens of the mask of  -min(r A, clip(r, low, high) A) + kl (exp(d) - 1 - d)
//   d loss / d z = c (onehot(t) - softmax(z)),  c = scale / M (-r A [not held by the clip] - kl (exp(d) - 1)).
// The coefficient c of a row depends on nothing but the row and M, so that the launch that reads a row for its log-sum-exp
// writes its gradient too, for a gradient of the loss of one; the backward has nothing left to do then but to look at that value.
#include "policy_loss.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int PL_THREADS = 1024;
constexpr int PL_WAVES = PL_THREADS / 64;

// 16-bit logits: the hardware's exponential (2^-21 relative at arguments of -20); 32-bit ones: the library's
template <typename IO> __device__ __forceinline__ float exp_of(float v) { return sizeof(IO) == 2 ? __expf(v) : expf(v); }

__device__ __forceinline__ float wave_max(float v) {
    for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
    return v;
}

// number of tokens that count -> 1 / M (M at least 1)
__global__ __launch_bounds__(PL_THREADS) void policy_count_kernel(const uint8_t *mask, int64_t N, float *inverse) {
    __shared__ int64_t parts[PL_WAVES];
    int64_t n = 0;
    for (int64_t i = threadIdx.x; i < N; i += PL_THREADS) n += mask == nullptr || mask[i] != 0;
    for (int m = 1; m < 64; m <<= 1) n += __shfl_xor(n, m, 64);
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < PL_WAVES; ++i) n += parts[i];
        *inverse = 1.0f / (float)(n > 0 ? n : 1);
    }
}

struct TokenTerms {
    float loss, coef;
};
// one token's share of the loss and its row's coefficient, both without scale / M
__device__ __forceinline__ TokenTerms terms_of(const PolicyLossArgs &a, int64_t row, float logp) {
    const float adv = a.adv[row], r = expf(logp - a.old_logp[row]), d = a.ref_logp[row] - logp, em = expm1f(d);
    const float freely = r * adv, held = fminf(fmaxf(r, a.low), a.high) * adv;
    const bool moves = freely < held || (r >= a.low && r <= a.high) || r != r;
    // the clip's comparisons drop a NaN that the sums keep
    return {(r != r ? r : -fminf(freely, held)) + a.kl * (em - d), (moves ? -freely : 0.0f) - a.kl * em};
}

// d z of a row, or its zeros
template <typename IO>
__device__ __forceinline__ void write_gradient(const IO *z, IO *dz, int64_t V, float lse, float c, int64_t target) {
    constexpr int VEC = 16 / sizeof(IO);
    for (int64_t i = (int64_t)threadIdx.x * VEC; i < V; i += PL_THREADS * VEC) {
        if (i + VEC <= V) {
            const Vec<IO, VEC> v = load_vec<IO, VEC>(z + i);
            Vec<IO, VEC> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float p = c == 0.0f ? 0.0f : -c * exp_of<IO>(widen(v.e[j]) - lse);
                o.e[j] = narrow<IO>(i + j == target ? p + c : p);
            }
            store_vec(dz + i, o);
        } else {
            for (int64_t j = i; j < V; ++j) {
                const float p = c == 0.0f ? 0.0f : -c * exp_of<IO>(widen(z[j]) - lse);
                dz[j] = narrow<IO>(j == target ? p + c : p);
            }
        }
    }
}

template <typename IO>
__global__ __launch_bounds__(PL_THREADS) void policy_rows_kernel(PolicyLossArgs a, const float *inverse) {
    constexpr int VEC = 16 / sizeof(IO);
    __shared__ float tops[PL_WAVES], sums[PL_WAVES], shared[2];
    const int64_t row = blockIdx.x;
    const IO *z = static_cast<const IO *>(a.logits) + row * a.V;
    float top = -INFINITY, s = 0;
    for (int64_t i = (int64_t)threadIdx.x * VEC; i < a.V; i += PL_THREADS * VEC) {
        float v[VEC];
        if (i + VEC <= a.V) {
            const Vec<IO, VEC> raw = load_vec<IO, VEC>(z + i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = widen(raw.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = i + j < a.V ? (float)widen(z[i + j]) : -INFINITY;
        }
        float m = top;
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = fmaxf(m, v[j]);
        const float base = m == -INFINITY ? 0.0f : m;
        s *= exp_of<IO>(top - base);
        top = m;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += exp_of<IO>(v[j] - base);
    }
    const float wm = wave_max(top), wbase = wm == -INFINITY ? 0.0f : wm;
    s = group_sum(s * exp_of<IO>(top - wbase), 64);
    if (threadIdx.x % 64 == 0) {
        tops[threadIdx.x / 64] = wm;
        sums[threadIdx.x / 64] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float m = tops[0];
        for (int i = 1; i < PL_WAVES; ++i) m = fmaxf(m, tops[i]);
        const float base = m == -INFINITY ? 0.0f : m;
        float total = 0;
        for (int i = 0; i < PL_WAVES; ++i) total += sums[i] * expf(tops[i] - base);
        const float lse = base + logf(total);
        const int64_t t = a.targets[row];
        const bool counts = a.mask == nullptr || a.mask[row] != 0, known = t >= 0 && t < a.V;
        const float logp = known ? widen(z[t]) - lse : counts ? NAN : 0.0f;
        const float share = a.scale * *inverse;
        TokenTerms m2{0, 0};
        if (counts) m2 = terms_of(a, row, logp);
        a.logp[row] = logp;
        a.lse[row] = shared[0] = lse;
        a.coef[row] = shared[1] = m2.coef * share;
        a.each[row] = m2.loss * share;
    }
    __syncthreads();
    if (a.d_logits != nullptr) write_gradient(z, static_cast<IO *>(a.d_logits) + row * a.V, a.V, shared[0], shared[1], a.targets[row]);
}

__global__ __launch_bounds__(PL_THREADS) void policy_sum_kernel(const float *each, int64_t N, float *loss) {
    __shared__ double parts[PL_WAVES];
    double s = 0;
    for (int64_t i = threadIdx.x; i < N; i += PL_THREADS) s += (double)each[i];
    s = group_sum(s, 64);
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < PL_WAVES; ++i) s += parts[i];
        *loss = (float)s;
    }
}

template <typename IO>
__global__ __launch_bounds__(PL_THREADS) void policy_gradient_kernel(PolicyLossArgs a) {
    const float g = *a.g_loss;
    if (a.unless_one && g == 1.0f) return;
    const int64_t row = blockIdx.x;
    const IO *z = static_cast<const IO *>(a.logits) + row * a.V;
    write_gradient(z, static_cast<IO *>(a.d_logits) + row * a.V, a.V, a.lse[row], a.coef[row] * g, a.targets[row]);
}

template <typename IO> int forward_of(const PolicyLossArgs &a, hipStream_t stream) {
    // 1 / M lies behind the tokens' shares
    float *const inverse = a.each + a.N;
    hipLaunchKernelGGL(policy_count_kernel, dim3(1), dim3(PL_THREADS), 0, stream, a.mask, a.N, inverse);
    int rc = check_hip(hipGetLastError(), "policy_count_kernel launch");
    if (rc) return rc;
    if (a.N > 0) {
        hipLaunchKernelGGL(policy_rows_kernel<IO>, dim3((unsigned)a.N), dim3(PL_THREADS), 0, stream, a, inverse);
        if ((rc = check_hip(hipGetLastError(), "policy_rows_kernel launch"))) return rc;
    }
    hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(PL_THREADS), 0, stream, a.each, a.N, a.loss);
    return check_hip(hipGetLastError(), "policy_sum_kernel launch");
}

template <typename IO> int backward_of(const PolicyLossArgs &a, hipStream_t stream) {
    if (a.N == 0) return T2FW_OK;
    hipLaunchKernelGGL(policy_gradient_kernel<IO>, dim3((unsigned)a.N), dim3(PL_THREADS), 0, stream, a);
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
