// Beam search: the best continuations over all beams of a request and the vocabulary, and the states of its beams moved to where they go on.
//
// Selection.  A candidate (k, v) has the score score_k + z_kv - lse_k.  Within a beam the logit alone orders candidates, so a workgroup reads a
// piece of 2048 to 16384 logits of one beam once, for its part of the log-sum-exp and for its n best; a second launch puts the parts together, in
// double, and takes the n best of all lists.  No two candidates are equal: of equal scores the lower beam, the larger logit and the lower token are better.
//   The n best of what 256 threads hold: n of the threads' largest are no smaller than the n-th largest of those, so nothing smaller can be among the n
//   best.  What is not smaller (most often little more than n, at most what n threads hold) goes to a list, where each counts those above it: its place.
//   The order in which the list is filled does not matter.
// Bound by memory for many logits, by latency for few: loads, five barriers a launch, two launches.
//
// Reordering.  A thread has the same 16 bytes of all beams of a request, loads those that move, and stores them when all of them are there: in place
// without a copy, and a beam that goes on from itself is neither read nor written.  One launch for up to 96 arrays.
#include <type_traits>
#include "beam.hpp"
#include "vec.hpp"

namespace t2fw {
namespace {

constexpr int THREADS = 256;
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

// A logit and its place in the piece, of 2^14 at most: 16 bits of both are enough for 16-bit logits.  All keys are larger than THREADS.
template <typename IO> struct Piece {
    typedef uint32_t Key;
    static __device__ __forceinline__ Key key(float z, uint32_t v) {
        const uint32_t u = __builtin_bit_cast(uint16_t, narrow<IO>(z + 0.0f));
        return (u & 0x8000u ? ~u << 16 : (u | 0x8000u) << 16) | (0xffffu - v);
    }
    static __device__ __forceinline__ float logit(Key k) {
        const uint16_t u = (uint16_t)(k >> 16);
        return widen(__builtin_bit_cast(IO, (uint16_t)(u & 0x8000u ? u & 0x7fffu : ~u)));
    }
    static __device__ __forceinline__ uint32_t place(Key k) { return 0xffffu - (k & 0xffffu); }
};
template <> struct Piece<float> {
    typedef uint64_t Key;
    static __device__ __forceinline__ Key key(float z, uint32_t v) { return packed(z, v); }
    static __device__ __forceinline__ float logit(Key k) { return logit_of(k); }
    static __device__ __forceinline__ uint32_t place(Key k) { return token_of(k); }
};

// A candidate of a request: its score, and what decides between equal ones, from the upper bits on: its beam (the lower is better), its logit and its token.
// Scores of one beam may be equal where its logits are not, as the sum next to a large score has no room for what sets them apart: the logit counts
// then, as in the choice of a piece's best.  Beams and tokens have 32 bits together.
struct Candidate {
    uint64_t key, next;
    __device__ __forceinline__ bool above(const Candidate &o) const { return key > o.key || (key == o.key && next > o.next); }
};
struct Ties {
    int bits;                                             // of a token
    __device__ __forceinline__ uint32_t tokens() const { return (1u << bits) - 1; }
    __device__ __forceinline__ uint64_t next(uint32_t k, uint32_t z, uint32_t v) const {
        return ~(uint64_t)k << (32 + bits) | (uint64_t)z << bits | (~v & tokens());
    }
    __device__ __forceinline__ uint32_t beam(uint64_t next) const { return (uint32_t)(~next >> (32 + bits)); }
    __device__ __forceinline__ uint32_t token(uint64_t next) const { return ~(uint32_t)next & tokens(); }
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

__device__ __forceinline__ uint32_t shuffled(uint32_t v, int m) { return __shfl_xor(v, m, 64); }
__device__ __forceinline__ uint64_t shuffled(uint64_t v, int m) { return __shfl_xor(v, m, 64); }
__device__ __forceinline__ Candidate shuffled(const Candidate &v, int m) { return {__shfl_xor(v.key, m, 64), __shfl_xor(v.next, m, 64)}; }

struct Share {
    float top;
    uint32_t unused;
    double sum;
};

// Groups of threads that the n best are looked for among: few, as each is compared with all, but some times n, or most groups are not below the n-th
__host__ __device__ constexpr int groups_of(int n) { return n <= 16 ? 64 : n <= 48 ? 128 : THREADS; }
// The best of a thread's group
template <typename Key, typename Above> __device__ __forceinline__ Key of_group(Key mine, int n, Above above) {
    if (n <= 48) {
        const Key o = shuffled(mine, 1);
        if (above(o, mine)) mine = o;
    }
    if (n <= 16) {
        const Key o = shuffled(mine, 2);
        if (above(o, mine)) mine = o;
    }
    return mine;
}
// How many of m numbers are above one: `per` (1, 2 or 4) threads side by side share them out, and all have the answer.  A loop of 64 took 1 us of the second launch.
template <typename Key, typename Above> __device__ __forceinline__ int count_above(const Key *all, int m, const Key &one, int per, Above above) {
    int place = 0;
#pragma unroll 8
    for (int i = threadIdx.x % per; i < m; i += per) place += above(all[i], one);
    if (per > 1) place += __shfl_xor(place, 1, 64);
    if (per > 2) place += __shfl_xor(place, 2, 64);
    return place;
}
__device__ __forceinline__ int threads_for(int m) { return m <= THREADS / 4 ? 4 : m <= THREADS / 2 ? 2 : 1; }
// The n-th largest of the groups' best, `mine`: all are distinct
template <typename Key, typename Above> __device__ __forceinline__ Key nth_best(const Key &mine, Key (&best)[THREADS], Key &least, int n, Above above) {
    const int groups = groups_of(n), per = THREADS / groups;
    if (threadIdx.x % per == 0) best[threadIdx.x / per] = mine;
    __syncthreads();
    const Key one = best[threadIdx.x / per];
    if (count_above(best, groups, one, per, above) == n - 1) least = one;      // (of each of its threads)
    __syncthreads();
    return least;
}

template <typename IO, int EACH> __global__ __launch_bounds__(THREADS) void beam_piece_kernel(BeamArgs a) {
    constexpr int VEC = 16 / sizeof(IO), VECS = EACH / VEC;
    __shared__ float tops[THREADS / 64];
    __shared__ double sums[THREADS / 64];
    typedef Piece<IO> Of;
    typedef typename Of::Key Key;
    __shared__ Key best[THREADS], least;
    __shared__ int found;
    extern __shared__ uint64_t memory[];
    Key *const list = reinterpret_cast<Key *>(memory);    // what the groups of threads that are not below the n-th hold
    const int64_t row = blockIdx.x / a.pieces;
    const int piece = blockIdx.x % a.pieces;
    const int64_t begin = (int64_t)piece * a.piece;
    const int here = a.V - begin < a.piece ? (int)(a.V - begin) : a.piece;
    const IO *const z = static_cast<const IO *>(a.logits) + row * a.V + begin;
    uint64_t *const to = a.lists + (int64_t)blockIdx.x * a.n;
    const bool ended = a.finished != nullptr && a.finished[row] != 0;
    if (ended || !(a.scores[row] > -INFINITY)) {
        // an ended beam has one candidate, the token for that, one that cannot be has none: then the others by their index
        const int pad = ended && a.pad >= begin && a.pad < begin + here ? (int)(a.pad - begin) : -1;
        for (int j = threadIdx.x; j < a.n; j += THREADS) {
            const int at = pad < 0 ? j : j == 0 ? pad : j <= pad ? j - 1 : j;
            to[j] = at < here ? packed(at == pad ? 0.0f : -INFINITY, (uint32_t)(begin + at)) : 0;
        }
        if (threadIdx.x == 0) static_cast<Share *>(a.partial)[blockIdx.x] = {-INFINITY, 0, 0.0};
        return;
    }
    // all loads at once, of what is not there of the first logits; the last vector of the piece, where it is no whole one, by its elements
    constexpr uint32_t NONE = sizeof(IO) == 4 ? 0xff800000u : std::is_same<IO, _Float16>::value ? 0xfc00fc00u : 0xff80ff80u;      // minus infinity
    uint32_t raw[VECS][4];
    if (here >= VEC) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int at = (i * THREADS + threadIdx.x) * VEC;
            const Vec<IO, VEC> one = load_vec<IO, VEC>(z + (at + VEC <= here ? at : 0));
            __builtin_memcpy(raw[i], &one, 16);
        }
    }
    float v[EACH];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const bool whole = (int)(i * THREADS + threadIdx.x) * VEC + VEC <= here;
#pragma unroll
        for (int w = 0; w < 4; ++w) raw[i][w] = whole ? raw[i][w] : NONE;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i * VEC + e] = element_of<IO>(raw[i], e);
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const int at = (i * THREADS + threadIdx.x) * VEC;
        if (at < here && at + VEC > here) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i * VEC + e] = at + e < here ? widen(z[at + e]) : -INFINITY;
        }
    }
    if (threadIdx.x == 0) found = 0;
    // a thread's largest, the first of equal ones
    float mine_z = -INFINITY;
    int mine_i = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) mine_z = fmaxf(mine_z, v[i]);
#pragma unroll
    for (int i = EACH - 1; i >= 0; --i) mine_i = v[i] == mine_z ? i : mine_i;
    const float top = over_group(mine_z, tops, [](float x, float y) { return fmaxf(x, y); });
    // Exponentials by the hardware, as powers of two: off by 2^-22, and by |z - top| 2^-23 for the exponent's rounding where e^(z - top) is the smaller.  Of
    // nothing above minus infinity the sum is zero, or NaN where there is one, which the largest does not show.
    // The difference and the product in one: what rounding the largest's product leaves is in all terms alike, and comes out of their sum again.
    constexpr float LOG2E = 1.44269504088896340736f;
    const float scaled = top * LOG2E, back = fabsf(top) < 0x1p20f ? fmaf(top, LOG2E, -scaled) : 0.0f;
    float parts[4] = {0.0f, 0.0f, 0.0f, 0.0f};           // (four sums: fewer roundings one after another)
    if (__builtin_amdgcn_readfirstlane(fabsf(top) < 0x1p20f)) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) parts[i % 4] += __builtin_amdgcn_exp2f(fmaf(v[i], LOG2E, -scaled));
    } else if (top > -INFINITY) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) parts[i % 4] += __builtin_amdgcn_exp2f((v[i] - top) * LOG2E);
    } else {
#pragma unroll
        for (int i = 0; i < EACH; ++i) parts[i % 4] += v[i] == v[i] ? 0.0f : v[i];
    }
    const float sum = (parts[0] + parts[1]) + (parts[2] + parts[3]);
    const double all = over_group((double)sum, sums, [](double x, double y) { return x + y; });
    if (threadIdx.x == 0) static_cast<Share *>(a.partial)[blockIdx.x] = {top, 0, all * __builtin_amdgcn_exp2f(-back)};
    // Logits of minus infinity and NaN stay out of it: where there are fewer others than wanted, the first of them follow by their index.  (Threads
    // that hold nothing are told apart by small numbers.)
    const int mine_at = (mine_i / VEC * THREADS + threadIdx.x) * VEC + mine_i % VEC;
    const Key mine = mine_z > -INFINITY ? Of::key(mine_z, (uint32_t)mine_at) : THREADS - threadIdx.x;
    const auto more = [](Key x, Key y) { return x > y; };
    const Key limit = nth_best(of_group(mine, a.n, more), best, least, a.n, more);
    if (mine > THREADS && mine >= limit) {
        // (a branch for eight: most threads have one that counts)
        const float limit_z = limit > THREADS ? Of::logit(limit) : -3.4028234e38f;
#pragma unroll
        for (int i = 0; i < EACH; i += 8) {
            float most = v[i];
#pragma unroll
            for (int e = 1; e < 8; ++e) most = fmaxf(most, v[i + e]);
            if (!(most >= limit_z)) continue;
#pragma unroll
            for (int e = i; e < i + 8; ++e) {
                if (!(v[e] >= limit_z)) continue;
                const Key k = Of::key(v[e], (uint32_t)((e / VEC * THREADS + threadIdx.x) * VEC + e % VEC));
                if (k >= limit) list[atomicAdd(&found, 1)] = k;
            }
        }
    }
    __syncthreads();
    const int m = found;
    const int per = threads_for(m);
    for (int j = threadIdx.x / per; j < m; j += THREADS / per) {
        const Key k = list[j];
        const int place = count_above(list, m, k, per, more);
        if (place < a.n) to[place] = packed(Of::logit(k), (uint32_t)begin + Of::place(k));
    }
    if (m >= a.n) return;
    // fewer than n others: of the first 2 n tokens at least n - m are none of them
    for (int j = threadIdx.x; j < 2 * a.n; j += THREADS) {
        int place = m + j;
        for (int i = 0; i < m; ++i) {
            const uint32_t t = Of::place(list[i]);
            place = t == (uint32_t)j ? a.n : place - (t < (uint32_t)j);      // (it has its place, which is below m)
            if (t == (uint32_t)j) break;
        }
        if (place < a.n) to[place] = j < here ? packed(-INFINITY, (uint32_t)(begin + j)) : 0;
    }
}

// A request: the n best of its lists, in rounds of up to 256 HOLD candidates, each with the n best so far.  A thread has some that follow each other in a
// list, so that the lists' first ones are with many threads: their n-th best is no worse than few others (64 requests, 16 x 131072 logits, 32 candidates: with
// the same places of several lists to a thread 33 us, so 21).
template <int HOLD> __global__ __launch_bounds__(THREADS) void beam_merge_kernel(BeamArgs a, int lanes, Ties ties) {
    __shared__ double sums[BEAM_ROWS];                    // logarithms of the sums; the largest logits stay apart
    __shared__ float tops[BEAM_ROWS], scores[BEAM_ROWS];
    __shared__ bool ended[BEAM_ROWS];
    __shared__ Candidate best[THREADS], least;
    __shared__ int found;
    extern __shared__ uint64_t memory[];                  // what the groups of threads hold, and the n of the rounds before
    Candidate *const kept = reinterpret_cast<Candidate *>(memory), *const list = kept + a.n;
    const int64_t b = blockIdx.x;
    const uint32_t per_beam = (uint32_t)a.pieces * a.n, total = (uint32_t)a.K * per_beam;
    const uint32_t each = total < THREADS * HOLD ? (total + THREADS - 1) / THREADS : HOLD;
    uint64_t p[HOLD];
    const auto load = [&](uint32_t from) {
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const uint32_t j = from + threadIdx.x * each + i;
            p[i] = (uint32_t)i < each && j < total ? a.lists[b * total + j] : 0;
        }
    };
    load(0);
    // `lanes` threads for a beam's pieces
    for (int k = threadIdx.x / lanes; k < a.K; k += THREADS / lanes) {
        const Share *const s = static_cast<const Share *>(a.partial) + (b * a.K + k) * a.pieces;
        const int in = threadIdx.x % lanes;
        float top = -INFINITY, most = -INFINITY;
        double sum = 0.0;
        if (in < a.pieces) {
            top = most = s[in].top;
            sum = s[in].sum;
        }
        for (int q = in + lanes; q < a.pieces; q += lanes) {
            const float t = s[q].top;
            most = fmaxf(top, t);
            sum = (top > -INFINITY ? sum * exp((double)top - (double)most) : sum) + (t > -INFINITY ? s[q].sum * exp((double)t - (double)most) : s[q].sum);
            top = most;
        }
        for (int m = 1; m < lanes; m <<= 1) most = fmaxf(most, __shfl_xor(most, m, 64));
        if (top > -INFINITY) sum *= exp((double)top - (double)most);
        for (int m = 1; m < lanes; m <<= 1) sum += __shfl_xor(sum, m, 64);
        if (in == 0) {
            tops[k] = most;
            sums[k] = log(sum);
            scores[k] = a.scores[b * a.K + k];
            ended[k] = a.finished != nullptr && a.finished[b * a.K + k] != 0;
        }
    }
    for (int j = threadIdx.x; j < a.n; j += THREADS) kept[j] = {0, (uint64_t)(THREADS + j)};
    __syncthreads();
    for (uint32_t from = 0; from < total; from += THREADS * each) {
        if (from > 0) load(from);
        if (threadIdx.x == 0) found = 0;
        // those of the rounds before are with the first n threads; threads that hold nothing are told apart by their places
        Candidate all[HOLD + 1], mine{0, threadIdx.x};
        if ((int)threadIdx.x < a.n) mine = kept[threadIdx.x];
        all[HOLD] = mine;
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const uint32_t k = p[i] != 0 ? (from + threadIdx.x * each + i) / per_beam : 0;
            const float score = scores[k], z = logit_of(p[i]);
            double s = -(double)INFINITY;
            if (ended[k]) s = z == 0.0f && token_of(p[i]) == (uint32_t)a.pad ? (double)score : s;
            else if (z > -INFINITY && score > -INFINITY) s = (double)score + (((double)z - (double)tops[k]) - sums[k]);
            all[i] = {p[i] != 0 ? ordered(s) : 0, ties.next(k, s > -(double)INFINITY ? ordered(z) : 0, token_of(p[i]))};
            if (all[i].key != 0 && all[i].above(mine)) mine = all[i];
        }
        const auto more = [](const Candidate &x, const Candidate &y) { return x.above(y); };
        const Candidate limit = nth_best(of_group(mine, a.n, more), best, least, a.n, more);
        if (!limit.above(mine)) {
#pragma unroll
            for (int i = 0; i <= HOLD; ++i)
                if (all[i].key != 0 && !limit.above(all[i])) list[atomicAdd(&found, 1)] = all[i];
        }
        __syncthreads();
        const int m = found;
        const int per = threads_for(m);
        for (int j = threadIdx.x / per; j < m; j += THREADS / per) {
            const Candidate one = list[j];
            const int place = count_above(list, m, one, per, more);
            if (place < a.n) kept[place] = one;
        }
        __syncthreads();
    }
    for (int j = threadIdx.x; j < a.n; j += THREADS) {
        const Candidate one = kept[j];
        a.out_scores[b * a.n + j] = (float)number(one.key);
        a.out_beams[b * a.n + j] = ties.beam(one.next);
        a.out_tokens[b * a.n + j] = ties.token(one.next);
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

// Logits of a thread: 64 where there are workgroups enough all the same, as what a workgroup does for its n best takes as long as 30 of a thread's logits;
// of few logits 8 (4 x 8000 float32: 10 us with 32, 7 so)
int beam_each(int64_t rows, int64_t V, int64_t n) {
    const auto pieces = [&](int each) { return (V + each * THREADS - 1) / (each * THREADS); };
    if (rows * pieces(64) >= 512 && n <= 96) return 64;            // (the list has to fit 64 KB of shared memory)
    return V <= 64 * THREADS && rows * pieces(32) < 256 ? 8 : 32;
}
BeamPieces beam_pieces(int64_t B, int64_t K, int64_t V, int64_t n_best) {
    const int64_t most = (int64_t)beam_each(B * K, V, n_best) * THREADS, n = (V + most - 1) / most;
    return {(int32_t)n, (int32_t)(((V + n - 1) / n + 7) / 8 * 8)};       // of nearly equal size, and no more than `most`, which is whole eights
}

template <typename IO> int launch_pieces(const BeamArgs &a, unsigned groups, size_t held, hipStream_t stream) {
    const int each = beam_each(a.B * a.K, a.V, a.n);
    const unsigned list = (unsigned)(each * held * sizeof(typename Piece<IO>::Key));
    if (each == 64) hipLaunchKernelGGL((beam_piece_kernel<IO, 64>), dim3(groups), dim3(THREADS), list, stream, a);
    else if (each == 32) hipLaunchKernelGGL((beam_piece_kernel<IO, 32>), dim3(groups), dim3(THREADS), list, stream, a);
    else hipLaunchKernelGGL((beam_piece_kernel<IO, 8>), dim3(groups), dim3(THREADS), list, stream, a);
    return check_hip(hipGetLastError(), "beam_piece_kernel launch");
}

int beam_select(const BeamArgs &a, int dtype, hipStream_t stream) {
    const int64_t groups = a.B * a.K * a.pieces;
    if (groups > MOST_GROUPS || a.B > MOST_GROUPS) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: too many workgroups for one launch");
    // threads of the n groups that are not below the n-th
    const int held = a.n * (THREADS / groups_of(a.n));
    const int hold = (int64_t)a.K * a.pieces * a.n <= 4 * THREADS ? 4 : 16;
    const unsigned merge = (unsigned)(((hold + 1) * held + a.n) * sizeof(Candidate));
    Ties ties{0};
    while (1ll << ties.bits < a.V) ++ties.bits;
    int lanes = 1;
    while (lanes < a.pieces && lanes < 64) lanes *= 2;
    const int rc = dtype == T2FW_F32 ? launch_pieces<float>(a, (unsigned)groups, held, stream) : dtype == T2FW_F16 ? launch_pieces<_Float16>(a, (unsigned)groups, held, stream) :
                   launch_pieces<__bf16>(a, (unsigned)groups, held, stream);
    if (rc) return rc;
    if (hold == 4) hipLaunchKernelGGL(beam_merge_kernel<4>, dim3((unsigned)a.B), dim3(THREADS), merge, stream, a, lanes, ties);
    else hipLaunchKernelGGL(beam_merge_kernel<16>, dim3((unsigned)a.B), dim3(THREADS), merge, stream, a, lanes, ties);
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
