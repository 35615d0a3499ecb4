// Beam search: the best continuations over all beams of a request and the vocabulary, and the states of its beams moved to where they go on.
//
// Selection.  A candidate (k, v) has the score score_k + z_kv - lse_k.  Within a beam the logit alone orders candidates, so a workgroup reads a
// piece of 8192 logits of one beam once, for its part of the log-sum-exp and for its n best; a second launch puts the parts together, in
// double, and takes the n best of all lists.  No two candidates are equal: of equal scores the lower index is the better one.
//   The n best of what 256 threads hold: n of the threads' largest are no smaller than the n-th largest of those, so nothing smaller can be among the n
//   best.  What is not smaller (most often little more than n, at most what n threads hold) goes to a list, where each counts those above it: its place.
//   The order in which the list is filled does not matter.
// Bound by memory for many logits, by latency for few: loads, three barriers, two launches.
//
// Reordering.  A thread has the same 16 bytes of all beams of a request, loads those that move, and stores them when all of them are there: in place
// without a copy, and a beam that goes on from itself is neither read nor written.  One launch for up to 96 arrays.
#include "beam.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int THREADS = 256, EACH = BEAM_PIECE / THREADS;
constexpr int64_t MOST_GROUPS = (1ll << 32) / THREADS - 1;      // a grid has less than 2^32 threads along an axis

// ---- keys ---------------------------------------------------------------------------------------------------------
// Numbers as unsigned ones of the same order, 0 less than any of them; NaN as minus infinity
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v == v ? v + 0.0f : -INFINITY);          // (+ 0: of the zeros the positive one)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float number(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v == v ? v + 0.0 : -(double)INFINITY);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double number(uint64_t k) { return __longlong_as_double((int64_t)(k >> 63 ? k & ~(1ull << 63) : ~k)); }

// A logit and its place in the beam in one number
__device__ __forceinline__ uint64_t packed(float z, uint32_t v) { return (uint64_t)ordered(z) << 32 | (0xffffffffu - v); }
__device__ __forceinline__ float logit_of(uint64_t p) { return number((uint32_t)(p >> 32)); }
__device__ __forceinline__ uint32_t token_of(uint64_t p) { return 0xffffffffu - (uint32_t)p; }

// A candidate of a request: its score, and its place among the K V
struct Candidate {
    uint64_t key;
    uint32_t at;
    __device__ __forceinline__ bool above(const Candidate &o) const { return key > o.key || (key == o.key && at < o.at); }
};

// ---- sums over a workgroup ----------------------------------------------------------------------------------------
template <typename T, typename Op> __device__ __forceinline__ T over_group(T v, T (&parts)[THREADS / 64], Op op) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = op(v, __shfl_xor(v, m, 64));
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = v;
    __syncthreads();
    v = parts[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) v = op(v, parts[i]);
    return v;
}

struct Share {
    float top;
    uint32_t unused;
    double sum;
};

template <typename IO> __global__ __launch_bounds__(THREADS) void beam_piece_kernel(BeamArgs a) {
    constexpr int VEC = 16 / sizeof(IO), VECS = EACH / VEC;
    __shared__ float tops[THREADS / 64];
    __shared__ double sums[THREADS / 64];
    __shared__ uint64_t best[THREADS], least;
    __shared__ int found;
    extern __shared__ uint64_t list[];                    // EACH n
    const int64_t row = blockIdx.x / a.pieces;
    const int piece = blockIdx.x % a.pieces;
    const int64_t begin = (int64_t)piece * BEAM_PIECE;
    const int here = a.V - begin < BEAM_PIECE ? (int)(a.V - begin) : BEAM_PIECE;
    const IO *const z = static_cast<const IO *>(a.logits) + row * a.V + begin;
    const bool ended = a.finished != nullptr && a.finished[row] != 0, never = !(a.scores[row] > -INFINITY);
    float v[EACH];
    if (ended || never) {
        // an ended beam has one candidate, the token for that; one that cannot be has none
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = (i / VEC * THREADS + threadIdx.x) * VEC + i % VEC;
            v[i] = ended && begin + at == a.pad ? 0.0f : -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int at = (i * THREADS + threadIdx.x) * VEC;
            if (at + VEC <= here) {
                const Vec<IO, VEC> x = load_vec<IO, VEC>(z + at);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i * VEC + e] = widen(x.e[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i * VEC + e] = at + e < here ? widen(z[at + e]) : -INFINITY;
            }
        }
    }
    if (threadIdx.x == 0) found = 0;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EACH; ++i) top = fmaxf(top, v[i]);
    top = over_group(top, tops, [](float x, float y) { return fmaxf(x, y); });
    float sum = 0.0f;
    if (top > -INFINITY) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) sum += expf(v[i] - top);
    } else {
        // nothing above minus infinity: nothing, or NaN that the largest does not show
#pragma unroll
        for (int i = 0; i < EACH; ++i) sum += v[i] == v[i] ? 0.0f : v[i];
    }
    const double all = over_group((double)sum, sums, [](double x, double y) { return x + y; });
    if (threadIdx.x == 0) static_cast<Share *>(a.partial)[blockIdx.x] = {top, 0, all};
    // the threads' best, and the n-th of those
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int at = (i / VEC * THREADS + threadIdx.x) * VEC + i % VEC;
        const uint64_t k = at < here ? packed(v[i], (uint32_t)(begin + at)) : 0;
        mine = k > mine ? k : mine;
    }
    best[threadIdx.x] = mine;
    __syncthreads();
    // (threads that hold nothing are told apart by their numbers)
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < THREADS; ++i) above += best[i] > mine || (best[i] == mine && i < (int)threadIdx.x);
    if (above == a.n - 1) least = mine;
    __syncthreads();
    const uint64_t limit = least > 0 ? least : 1;
    if (mine >= limit) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = (i / VEC * THREADS + threadIdx.x) * VEC + i % VEC;
            const uint64_t k = at < here ? packed(v[i], (uint32_t)(begin + at)) : 0;
            if (k >= limit) list[atomicAdd(&found, 1)] = k;
        }
    }
    __syncthreads();
    uint64_t *const to = a.lists + (int64_t)blockIdx.x * a.n;
    const int m = found;
    for (int j = threadIdx.x; j < m; j += THREADS) {
        const uint64_t k = list[j];
        int place = 0;
        for (int i = 0; i < m; ++i) place += list[i] > k;
        if (place < a.n) to[place] = k;
    }
    for (int j = m + threadIdx.x; j < a.n; j += THREADS) to[j] = 0;      // fewer logits than that
}

// A request: the n best of its lists, in rounds of ROUND candidates, each with the n best so far
constexpr int HOLD = 8, ROUND = THREADS * HOLD;
__global__ __launch_bounds__(THREADS) void beam_merge_kernel(BeamArgs a) {
    __shared__ double lse[BEAM_ROWS];                     // (the largest logit and the logarithm of the sum apart, as they are added)
    __shared__ float tops[BEAM_ROWS];
    __shared__ Candidate best[THREADS], least;
    __shared__ int found;
    extern __shared__ uint64_t memory[];                  // (HOLD + 1) n candidates, and n of the rounds before
    Candidate *const list = reinterpret_cast<Candidate *>(memory), *const kept = list + (HOLD + 1) * a.n;
    const int64_t b = blockIdx.x;
    const uint32_t per_beam = (uint32_t)a.pieces * a.n, total = (uint32_t)a.K * per_beam;
    for (int k = threadIdx.x; k < a.K; k += THREADS) {
        const Share *const s = static_cast<const Share *>(a.partial) + (b * a.K + k) * a.pieces;
        float top = -INFINITY;
        for (int p = 0; p < a.pieces; ++p) top = fmaxf(top, s[p].top);
        double sum = 0.0;
        for (int p = 0; p < a.pieces; ++p) sum += s[p].top > -INFINITY ? s[p].sum * exp((double)s[p].top - (double)top) : s[p].sum;
        tops[k] = top;
        lse[k] = log(sum);
    }
    for (int j = threadIdx.x; j < a.n; j += THREADS) kept[j] = {0, 0xffffffffu};
    __syncthreads();
    for (uint32_t from = 0; from < total; from += ROUND) {
        if (threadIdx.x == 0) found = 0;
        // those of the rounds before are with the first n threads
        uint64_t key[HOLD + 1];
        uint32_t at[HOLD + 1];
        Candidate mine{0, 0xffffffffu};
        if ((int)threadIdx.x < a.n) mine = kept[threadIdx.x];
        key[HOLD] = mine.key;
        at[HOLD] = mine.at;
        uint64_t p[HOLD];
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const uint32_t j = from + i * THREADS + threadIdx.x;
            p[i] = j < total ? a.lists[b * total + j] : 0;
        }
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const uint32_t j = from + i * THREADS + threadIdx.x, k = p[i] != 0 ? j / per_beam : 0;
            const float score = a.scores[b * a.K + k], z = logit_of(p[i]);
            double s = -(double)INFINITY;
            if (a.finished != nullptr && a.finished[b * a.K + k] != 0) s = z == 0.0f && token_of(p[i]) == (uint32_t)a.pad ? (double)score : s;
            else if (z > -INFINITY && score > -INFINITY) s = (double)score + (((double)z - (double)tops[k]) - lse[k]);
            key[i] = p[i] != 0 ? ordered(s) : 0;
            at[i] = p[i] != 0 ? k * (uint32_t)a.V + token_of(p[i]) : 0xffffffffu;
            const Candidate one{key[i], at[i]};
            if (one.above(mine)) mine = one;
        }
        best[threadIdx.x] = mine;
        __syncthreads();
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < THREADS; ++i) above += best[i].above(mine) || (!mine.above(best[i]) && i < (int)threadIdx.x);
        if (above == a.n - 1) least = mine;
        __syncthreads();
        const Candidate limit = least;
#pragma unroll
        for (int i = 0; i <= HOLD; ++i) {
            const Candidate one{key[i], at[i]};
            if (one.key != 0 && !limit.above(one)) list[atomicAdd(&found, 1)] = one;
        }
        __syncthreads();
        const int m = found;
        for (int j = threadIdx.x; j < m; j += THREADS) {
            const Candidate one = list[j];
            int place = 0;
            for (int i = 0; i < m; ++i) place += list[i].above(one);
            if (place < a.n) kept[place] = one;
        }
        __syncthreads();
    }
    for (int j = threadIdx.x; j < a.n; j += THREADS) {
        const Candidate one = kept[j];
        a.out_scores[b * a.n + j] = (float)number(one.key);
        a.out_beams[b * a.n + j] = one.at / (uint32_t)a.V;
        a.out_tokens[b * a.n + j] = one.at % (uint32_t)a.V;
    }
}

// ---- reordering ---------------------------------------------------------------------------------------------------
// (at any byte: global memory takes unaligned accesses)
struct Word16 {
    typedef uint32_t Held __attribute__((ext_vector_type(4)));
    typedef uint32_t There __attribute__((ext_vector_type(4), aligned(1)));
    static constexpr int BYTES = 16;
    static __device__ __forceinline__ Held load(const char *p) { return *reinterpret_cast<const There *>(p); }
    static __device__ __forceinline__ void store(char *p, Held v) { *reinterpret_cast<There *>(p) = v; }
};
struct Word4 {
    typedef uint32_t Held;
    typedef uint32_t There __attribute__((aligned(1)));
    static constexpr int BYTES = 4;
    static __device__ __forceinline__ Held load(const char *p) { return *reinterpret_cast<const There *>(p); }
    static __device__ __forceinline__ void store(char *p, Held v) { *reinterpret_cast<There *>(p) = v; }
};
struct Word1 {
    typedef uint8_t Held;
    static constexpr int BYTES = 1;
    static __device__ __forceinline__ Held load(const char *p) { return *reinterpret_cast<const uint8_t *>(p); }
    static __device__ __forceinline__ void store(char *p, Held v) { *reinterpret_cast<uint8_t *>(p) = v; }
};
// Word by word, the words of a piece dealt out to the threads
template <int K, typename Word>
__device__ __forceinline__ void move_words(const char *src, char *dst, int64_t row, int64_t begin, int64_t end, const int (&from)[K], int beams, bool in_place) {
    for (int64_t at = begin + (int64_t)threadIdx.x * Word::BYTES; at + Word::BYTES <= end; at += THREADS * Word::BYTES) {
        typename Word::Held held[K];
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < beams && (!in_place || from[k] != k)) held[k] = Word::load(src + from[k] * row + at);
        wait_vmem_all();                                 // (all of them, before the first place is written again)
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < beams && (!in_place || from[k] != k)) Word::store(dst + k * row + at, held[k]);
    }
}
template <int K, typename Word> __global__ __launch_bounds__(THREADS) void beam_reorder_kernel(ReorderTable t, const int64_t *beams, int64_t B, int K_, int64_t piece) {
    const uint32_t n = blockIdx.x;
    int lo = 0, hi = (int)t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= n) lo = mid;
        else hi = mid - 1;
    }
    const int64_t row = t.row[lo], per_request = (row + piece - 1) / piece, in = n - t.first[lo], b = in / per_request;
    const int64_t begin = (in - b * per_request) * piece, end = begin + piece < row ? begin + piece : row;
    const char *const src = t.src[lo] + b * K_ * row;
    char *const dst = t.dst[lo] + b * K_ * row;
    int from[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int64_t f = k < K_ ? beams[b * K_ + k] : k;
        from[k] = __builtin_amdgcn_readfirstlane((int)(f >= 0 && f < K_ ? f : k));       // (no such beam: the one that is there)
    }
    const int64_t whole = begin + (end - begin) / Word::BYTES * Word::BYTES;
    move_words<K, Word>(src, dst, row, begin, whole, from, K_, src == dst);
    move_words<K, Word1>(src, dst, row, whole, end, from, K_, src == dst);
}
template <int K, typename Word> int launch_reorder(const ReorderTable &t, const int64_t *beams, int64_t B, int64_t beams_of, hipStream_t stream) {
    hipLaunchKernelGGL((beam_reorder_kernel<K, Word>), dim3(t.pieces), dim3(THREADS), 0, stream, t, beams, B, (int)beams_of, reorder_piece(beams_of));
    return check_hip(hipGetLastError(), "beam_reorder_kernel launch");
}

}  // namespace

int beam_select(const BeamArgs &a, int dtype, hipStream_t stream) {
    const int64_t groups = a.B * a.K * a.pieces;
    if (groups > MOST_GROUPS || a.B > MOST_GROUPS) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: too many workgroups for one launch");
    const dim3 grid((unsigned)groups), threads(THREADS);
    const unsigned list = (unsigned)(EACH * a.n * sizeof(uint64_t)), merge = (unsigned)((HOLD + 2) * a.n * sizeof(Candidate));
    if (dtype == T2FW_F32) hipLaunchKernelGGL(beam_piece_kernel<float>, grid, threads, list, stream, a);
    else if (dtype == T2FW_F16) hipLaunchKernelGGL(beam_piece_kernel<_Float16>, grid, threads, list, stream, a);
    else hipLaunchKernelGGL(beam_piece_kernel<__bf16>, grid, threads, list, stream, a);
    int rc = check_hip(hipGetLastError(), "beam_piece_kernel launch");
    if (rc) return rc;
    hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)a.B), threads, merge, stream, a);
    return check_hip(hipGetLastError(), "beam_merge_kernel launch");
}

// 4 KB, a round of 16-byte words; of many beams a round of words that fit the registers
int64_t reorder_piece(int64_t K) { return K <= 16 ? THREADS * 16 : THREADS * 4; }

int beam_reorder(const ReorderTable &t, const int64_t *beams, int64_t B, int64_t K, hipStream_t stream) {
    if (K <= 4) return launch_reorder<4, Word16>(t, beams, B, K, stream);
    if (K <= 8) return launch_reorder<8, Word16>(t, beams, B, K, stream);
    if (K <= 16) return launch_reorder<16, Word16>(t, beams, B, K, stream);
    return launch_reorder<REORDER_BEAMS, Word4>(t, beams, B, K, stream);
}

}  // namespace t2fw
