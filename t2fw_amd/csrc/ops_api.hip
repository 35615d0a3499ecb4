// C ABI of the operators around the recurrences (include/t2fw_hip.h): argument validation, and what a call needs laid out.
#include "common.hpp"
#include "clip.hpp"
#include "gscan.hpp"
#include "policy_loss.hpp"
#include "rmsnorm.hpp"

#include <cmath>
#include <vector>

namespace t2fw {
namespace {

size_t size_of(int dtype) { return dtype == T2FW_F64 ? 8 : dtype == T2FW_F32 ? 4 : dtype == T2FW_F16 || dtype == T2FW_BF16 ? 2 : 0; }
size_t accumulator_size(int dtype) { return dtype == T2FW_F64 ? 8 : 4; }

int bad_dtype(int dtype) { return fail(T2FW_ERR_BAD_DTYPE, "unknown dtype code %d", dtype); }
int bad_workspace(size_t need, size_t given) { return fail(T2FW_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, given); }

struct Array {
    const char *name;
    const void *at;
    size_t align;
    bool optional;
};
int check_arrays(std::initializer_list<Array> arrays) {
    for (const Array &a : arrays) {
        if (a.at == nullptr) {
            if (a.optional) continue;
            return fail(T2FW_ERR_NULL_POINTER, "%s is a null pointer", a.name);
        }
        if (reinterpret_cast<uintptr_t>(a.at) % a.align != 0)
            return fail(T2FW_ERR_MISALIGNED, "%s is not aligned to %zu bytes", a.name, a.align);
    }
    return T2FW_OK;
}
// sizes whose product in bytes is addressable
int check_sizes(std::initializer_list<int64_t> sizes, const char *what) {
    long double bytes = 16;
    for (int64_t n : sizes) {
        if (n < 0) return fail(T2FW_ERR_BAD_SHAPE, "%s: sizes must be non-negative", what);
        bytes *= n > 0 ? (long double)n : 1;
    }
    if (bytes > 9.0e18L) return fail(T2FW_ERR_BAD_SHAPE, "%s: not addressable", what);
    return T2FW_OK;
}

// A look takes about a microsecond: what is not there after these has not been started, and its workgroup will be long in coming
constexpr int SCAN_LOOKS = 1 << 14;

int check_scan(int64_t B, int64_t T, int64_t D, int32_t dtype, int32_t flags) {
    if (size_of(dtype) == 0) return bad_dtype(dtype);
    const int rc = check_sizes({B, T, D}, "gated scan");
    if (rc) return rc;
    if (D < 1) return fail(T2FW_ERR_BAD_SHAPE, "gated scan: at least one channel");
    if (flags & ~(T2FW_SCAN_LOGITS | T2FW_SCAN_LENGTHS64 | T2FW_SCAN_ALONE)) return fail(T2FW_ERR_UNSUPPORTED, "gated scan: unknown flags %d", flags);
    return T2FW_OK;
}
int scan_strides(GscanArgs &a, const int64_t *strides, bool backward) {
    a.x_b = a.f_b = a.g_b = a.T * a.D;
    a.x_t = a.f_t = a.g_t = a.D;
    if (strides == nullptr) return T2FW_OK;
    for (int i = 0; i < (backward ? 6 : 4); ++i)
        if (strides[i] < 0) return fail(T2FW_ERR_BAD_SHAPE, "gated scan: strides must be non-negative");
    a.x_b = strides[0]; a.x_t = strides[1]; a.f_b = strides[2]; a.f_t = strides[3];
    if (backward) {
        a.g_b = strides[4]; a.g_t = strides[5];
    }
    return T2FW_OK;
}

int check_norm(int64_t N, int64_t D, int32_t dtype, int32_t flags) {
    if (size_of(dtype) == 0) return bad_dtype(dtype);
    const int rc = check_sizes({N, D}, "norm");
    if (rc) return rc;
    if (D < 1) return fail(T2FW_ERR_BAD_SHAPE, "norm: at least one column");
    if (flags & ~(T2FW_NORM_STREAM_F32 | T2FW_NORM_WEIGHT_F32)) return fail(T2FW_ERR_UNSUPPORTED, "norm: unknown flags %d", flags);
    if (flags != 0 && dtype == T2FW_F64) return fail(T2FW_ERR_UNSUPPORTED, "norm: float streams and weights go with 16-bit tensors");
    return T2FW_OK;
}
// what an array is aligned to that may be float next to 16-bit ones
size_t wide_size(int32_t dtype, bool wide) { return wide ? 4 : size_of(dtype); }
NormArgs norm_args(int64_t N, int64_t D, double eps, int32_t dtype, int32_t flags) {
    NormArgs a{};
    a.N = N; a.D = D; a.eps = eps;
    a.wide_stream = dtype != T2FW_F32 && (flags & T2FW_NORM_STREAM_F32) != 0;
    a.wide_w = dtype == T2FW_F32 || (flags & T2FW_NORM_WEIGHT_F32) != 0;
    return a;
}

int check_loss(int64_t N, int64_t V, int32_t dtype) {
    if (dtype != T2FW_F32 && dtype != T2FW_F16 && dtype != T2FW_BF16)
        return fail(T2FW_ERR_BAD_DTYPE, "the policy loss takes fp32, fp16 or bf16 logits (dtype code %d)", dtype);
    const int rc = check_sizes({N, V}, "policy loss");
    if (rc) return rc;
    if (V < 1) return fail(T2FW_ERR_BAD_SHAPE, "policy loss: at least one logit");
    if (N > 0x7fffffff) return fail(T2FW_ERR_BAD_SHAPE, "policy loss: too many tokens for one launch");
    return T2FW_OK;
}

// Arrays in tables of at most CLIP_TABLE entries of less than 2^32 elements; empty arrays left out
int clip_tables(std::vector<ClipTable> &tables, const t2fw_clip_desc *arrays, int64_t count) {
    if (count < 0 || count > 0x7fffffff) return fail(T2FW_ERR_BAD_SHAPE, "clipping: %lld arrays", (long long)count);
    if (count > 0 && arrays == nullptr) return fail(T2FW_ERR_NULL_POINTER, "null array list");
    constexpr int64_t MOST = (int64_t)CLIP_PIECE << 19;              // elements of one entry: 2^30, a whole number of pieces
    for (int64_t i = 0; i < count; ++i) {
        const t2fw_clip_desc &d = arrays[i];
        const size_t es = size_of(d.src_dtype), ed = size_of(d.dst_dtype);
        if (es == 0 || (d.dst != nullptr && ed == 0)) return bad_dtype(es == 0 ? d.src_dtype : d.dst_dtype);
        int rc = check_sizes({d.n}, "clipping");
        if (rc) return rc;
        if (d.n == 0) continue;
        if ((rc = check_arrays({{"src", d.src, es, false}, {"dst", d.dst, ed ? ed : 1, true}}))) return rc;
        if (d.dst == d.src && d.dst != nullptr && d.src_dtype != d.dst_dtype)
            return fail(T2FW_ERR_BAD_DTYPE, "clipping in place: the array has two types");
        for (int64_t at = 0; at < d.n; at += MOST) {
            if (tables.empty() || tables.back().count == CLIP_TABLE || tables.back().pieces > (1u << 30)) tables.push_back(ClipTable{});
            ClipTable &t = tables.back();
            const int64_t n = d.n - at < MOST ? d.n - at : MOST;
            t.src[t.count] = static_cast<const char *>(d.src) + at * es;
            t.dst[t.count] = d.dst == nullptr ? nullptr : static_cast<char *>(d.dst) + at * ed;
            t.n[t.count] = (uint32_t)n;
            t.first[t.count] = t.pieces;
            t.src_type[t.count] = (uint8_t)d.src_dtype;
            t.dst_type[t.count] = (uint8_t)d.dst_dtype;
            t.pieces += (uint32_t)((n + CLIP_PIECE - 1) / CLIP_PIECE);
            ++t.count;
        }
    }
    return T2FW_OK;
}
int clip_groups(const ClipTable &t) { return t.pieces < (uint32_t)CLIP_GROUPS ? (int)t.pieces : CLIP_GROUPS; }

}  // namespace
}  // namespace t2fw

using namespace t2fw;

extern "C" {

size_t t2fw_gated_scan_checkpoint_bytes(int64_t B, int64_t T, int64_t D, int32_t dtype) {
    if (check_scan(B, T, D, dtype, 0) || B == 0) return 0;
    return gscan_plan(B, T, D, dtype).checkpoints;
}

size_t t2fw_gated_scan_workspace_bytes(int64_t B, int64_t T, int64_t D, int32_t dtype) {
    if (check_scan(B, T, D, dtype, 0) || B == 0) return 0;
    return gscan_plan(B, T, D, dtype).workspace;
}

int t2fw_gated_scan_forward(const void *x, const void *f, const void *s0, const void *lengths, void *out, void *final_state, void *ckpt,
                            int64_t B, int64_t T, int64_t D, const int64_t *strides, int32_t dtype, int32_t flags, void *workspace,
                            size_t workspace_bytes, void *stream) {
    int rc = check_scan(B, T, D, dtype, flags);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    const size_t es = size_of(dtype), ac = accumulator_size(dtype), need = t2fw_gated_scan_workspace_bytes(B, T, D, dtype);
    if ((rc = check_arrays({{"x", x, es, T == 0}, {"f", f, es, T == 0}, {"out", out, es, T == 0}, {"s0", s0, ac, true},
                            {"final_state", final_state, ac, false}, {"ckpt", ckpt, 16, true},
                            {"lengths", lengths, flags & T2FW_SCAN_LENGTHS64 ? 8u : 4u, true}, {"workspace", workspace, 16, need == 0}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    GscanArgs a{};
    a.x = x; a.f = f; a.s0 = s0; a.lengths = lengths; a.out = out; a.final_state = final_state; a.ckpt = ckpt; a.words = workspace;
    a.B = B; a.T = T; a.D = D;
    a.logits = (flags & T2FW_SCAN_LOGITS) != 0;
    a.wide_lengths = (flags & T2FW_SCAN_LENGTHS64) != 0;
    a.looks = flags & T2FW_SCAN_ALONE ? 0 : SCAN_LOOKS;
    if ((rc = scan_strides(a, strides, false))) return rc;
    return gscan_forward(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_gated_scan_backward(const void *g_out, const void *g_state, const void *x, const void *f, const void *lengths, const void *ckpt,
                             void *d_x, void *d_f, void *d_s0, int64_t B, int64_t T, int64_t D, const int64_t *strides, int32_t dtype,
                             int32_t flags, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_scan(B, T, D, dtype, flags);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    const size_t es = size_of(dtype), ac = accumulator_size(dtype), need = t2fw_gated_scan_workspace_bytes(B, T, D, dtype);
    if ((rc = check_arrays({{"g_out", g_out, es, T == 0}, {"g_state", g_state, ac, true}, {"x", x, es, T == 0}, {"f", f, es, T == 0},
                            {"lengths", lengths, flags & T2FW_SCAN_LENGTHS64 ? 8u : 4u, true}, {"ckpt", ckpt, 16, false},
                            {"d_x", d_x, es, T == 0}, {"d_f", d_f, es, T == 0}, {"d_s0", d_s0, ac, true}, {"workspace", workspace, 16, need == 0}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    GscanArgs a{};
    a.g_out = g_out; a.g_state = g_state; a.x = x; a.f = f; a.lengths = lengths; a.ckpt = const_cast<void *>(ckpt);
    a.d_x = d_x; a.d_f = d_f; a.d_s0 = d_s0; a.words = workspace;
    a.B = B; a.T = T; a.D = D;
    a.logits = (flags & T2FW_SCAN_LOGITS) != 0;
    a.wide_lengths = (flags & T2FW_SCAN_LENGTHS64) != 0;
    a.looks = flags & T2FW_SCAN_ALONE ? 0 : SCAN_LOOKS;
    if ((rc = scan_strides(a, strides, true))) return rc;
    return gscan_backward(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_gated_scan_step(const void *x, const void *f, const void *s0, void *out, void *next_state, int64_t B, int64_t D, int32_t dtype,
                         int32_t flags, void *stream) {
    int rc = check_scan(B, 1, D, dtype, flags);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    const size_t es = size_of(dtype), ac = accumulator_size(dtype);
    if ((rc = check_arrays({{"x", x, es, false}, {"f", f, es, false}, {"s0", s0, ac, false}, {"out", out, es, false},
                            {"next_state", next_state, ac, false}})))
        return rc;
    GscanArgs a{};
    a.x = x; a.f = f; a.s0 = s0; a.out = out; a.final_state = next_state;
    a.B = B; a.T = 1; a.D = D;
    a.logits = (flags & T2FW_SCAN_LOGITS) != 0;
    return gscan_step(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_rms_norm_forward(const void *x, const void *res, const void *w, void *y, void *stored, int64_t N, int64_t D, double eps,
                          int32_t dtype, int32_t flags, void *stream) {
    int rc = check_norm(N, D, dtype, flags);
    if (rc) return rc;
    if (N == 0) return T2FW_OK;
    const size_t es = size_of(dtype), ss = wide_size(dtype, flags & T2FW_NORM_STREAM_F32), ws = wide_size(dtype, flags & T2FW_NORM_WEIGHT_F32);
    if ((rc = check_arrays({{"x", x, es, false}, {"res", res, ss, true}, {"w", w, ws, false}, {"y", y, es, false},
                            {"stored", stored, ss, res == nullptr}})))
        return rc;
    NormArgs a = norm_args(N, D, eps, dtype, flags);
    a.x = x; a.res = res; a.w = w; a.y = y; a.stored = stored;
    return norm_forward(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_rms_norm_forward_fp8(const void *x, const void *res, const void *w, void *q, float *scales, void *stored, int64_t N, int64_t D,
                              int64_t group, double eps, int32_t dtype, int32_t flags, void *stream) {
    int rc = check_norm(N, D, dtype, flags);
    if (rc) return rc;
    if (dtype == T2FW_F64) return fail(T2FW_ERR_BAD_DTYPE, "the norm in 8 bits takes fp32, fp16 or bf16");
    if (group != 0 && (group < 8 || group > 512 || (group & (group - 1)) != 0))
        return fail(T2FW_ERR_BAD_SHAPE, "columns of a scale: 0 (the row) or a power of two from 8 to 512, not %lld", (long long)group);
    if (N == 0) return T2FW_OK;
    const size_t es = size_of(dtype), ss = wide_size(dtype, flags & T2FW_NORM_STREAM_F32), ws = wide_size(dtype, flags & T2FW_NORM_WEIGHT_F32);
    if ((rc = check_arrays({{"x", x, es, false}, {"res", res, ss, true}, {"w", w, ws, false}, {"q", q, 1, false}, {"scales", scales, 4, false},
                            {"stored", stored, ss, res == nullptr}})))
        return rc;
    NormArgs a = norm_args(N, D, eps, dtype, flags);
    a.x = x; a.res = res; a.w = w; a.q = q; a.scales = scales; a.stored = stored;
    a.group = group;
    a.groups = group == 0 ? 1 : (D + group - 1) / group;
    return norm_forward(a, dtype, static_cast<hipStream_t>(stream));
}

size_t t2fw_rms_norm_backward_workspace_bytes(int64_t N, int64_t D, int32_t dtype) {
    if (check_norm(N, D, dtype, 0)) return 0;
    return (size_t)(norm_partials(N, D) * D) * accumulator_size(dtype);
}

int t2fw_rms_norm_backward(const void *g_y, const void *g_res, const void *stored, const void *w, void *d_x, void *d_res, void *d_w, int64_t N,
                           int64_t D, double eps, int32_t dtype, int32_t flags, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_norm(N, D, dtype, flags);
    if (rc) return rc;
    const size_t es = size_of(dtype), ss = wide_size(dtype, flags & T2FW_NORM_STREAM_F32), ws = wide_size(dtype, flags & T2FW_NORM_WEIGHT_F32);
    const size_t need = t2fw_rms_norm_backward_workspace_bytes(N, D, dtype);
    if ((rc = check_arrays({{"g_y", g_y, es, N == 0}, {"g_res", g_res, ss, true}, {"stored", stored, ss, N == 0}, {"w", w, ws, false},
                            {"d_x", d_x, es, N == 0}, {"d_res", d_res, ss, ss == es || N == 0}, {"d_w", d_w, ws, false},
                            {"workspace", workspace, 16, need == 0}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    NormArgs a = norm_args(N, D, eps, dtype, flags);
    a.g_y = g_y; a.g_res = g_res; a.stored = const_cast<void *>(stored); a.w = w; a.d_x = d_x; a.d_res = d_res; a.d_w = d_w;
    a.partials = workspace;
    return norm_backward(a, dtype, static_cast<hipStream_t>(stream));
}

size_t t2fw_policy_loss_workspace_bytes(int64_t N) { return N < 0 ? 0 : (POLICY_SUMS + 1) * sizeof(double); }

int t2fw_policy_loss_forward(const void *logits, const int64_t *targets, const float *old_logp, const float *ref_logp, const float *adv,
                             const void *mask, float *loss, float *logp, float *tops, float *coef, void *d_logits, int64_t N, int64_t V,
                             float low, float high, float kl, float scale, int32_t dtype, void *workspace, size_t workspace_bytes,
                             void *stream) {
    int rc = check_loss(N, V, dtype);
    if (rc) return rc;
    if (!(low <= high)) return fail(T2FW_ERR_BAD_SHAPE, "policy loss: ratios are held in [%g, %g]", (double)low, (double)high);
    const size_t es = size_of(dtype), need = t2fw_policy_loss_workspace_bytes(N);
    const bool none = N == 0;
    if ((rc = check_arrays({{"logits", logits, es, none}, {"targets", targets, 8, none}, {"old_logp", old_logp, 4, none},
                            {"ref_logp", ref_logp, 4, none}, {"adv", adv, 4, none}, {"loss", loss, 4, false}, {"logp", logp, 4, none},
                            {"tops", tops, 4, none}, {"coef", coef, 4, none}, {"d_logits", d_logits, es, true}, {"workspace", workspace, 8, false}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    PolicyLossArgs a{};
    a.logits = logits; a.targets = targets; a.old_logp = old_logp; a.ref_logp = ref_logp; a.adv = adv;
    a.mask = static_cast<const uint8_t *>(mask);
    a.loss = loss; a.logp = logp; a.tops = tops; a.coef = coef; a.tokens = static_cast<int64_t *>(workspace);
    a.sums = static_cast<double *>(workspace) + 1; a.d_logits = d_logits;
    a.N = N; a.V = V; a.low = low; a.high = high; a.kl = kl; a.scale = scale;
    return policy_loss_forward(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_policy_loss_backward(const void *logits, const int64_t *targets, const float *tops, const float *coef, const float *g_loss,
                              void *d_logits, int64_t N, int64_t V, int32_t dtype, int32_t flags, void *stream) {
    int rc = check_loss(N, V, dtype);
    if (rc) return rc;
    if (flags & ~T2FW_LOSS_UNLESS_ONE) return fail(T2FW_ERR_UNSUPPORTED, "policy loss: unknown flags %d", flags);
    if (N == 0) return T2FW_OK;
    const size_t es = size_of(dtype);
    if ((rc = check_arrays({{"logits", logits, es, false}, {"targets", targets, 8, false}, {"tops", tops, 4, false}, {"coef", coef, 4, false},
                            {"g_loss", g_loss, 4, false}, {"d_logits", d_logits, es, false}})))
        return rc;
    PolicyLossArgs a{};
    a.logits = logits; a.targets = targets; a.tops = const_cast<float *>(tops); a.coef = const_cast<float *>(coef); a.g_loss = g_loss;
    a.d_logits = d_logits;
    a.N = N; a.V = V;
    a.unless_one = (flags & T2FW_LOSS_UNLESS_ONE) != 0;
    return policy_loss_backward(a, dtype, static_cast<hipStream_t>(stream));
}

size_t t2fw_clip_workspace_bytes(const t2fw_clip_desc *arrays, int64_t count) try {
    std::vector<ClipTable> tables;
    if (clip_tables(tables, arrays, count)) return 0;
    size_t groups = 1;                               // at least one, for no arrays at all
    for (const ClipTable &t : tables) groups += clip_groups(t);
    return groups * sizeof(double);
} catch (const std::exception &) {
    return 0;
}

int t2fw_clip_grad_norm(const t2fw_clip_desc *arrays, int64_t count, float max_norm, float *norm, void *workspace, size_t workspace_bytes,
                        void *stream) {
    return t2fw_clip_grad_norm_f64(arrays, count, max_norm, norm, workspace, workspace_bytes, stream);
}

int t2fw_clip_grad_norm_f64(const t2fw_clip_desc *arrays, int64_t count, double max_norm, float *norm, void *workspace, size_t workspace_bytes,
                            void *stream) try {
    std::vector<ClipTable> tables;
    int rc = clip_tables(tables, arrays, count);
    if (rc) return rc;
    if (!(max_norm >= 0)) return fail(T2FW_ERR_BAD_SHAPE, "clipping: a largest norm of %g", max_norm);
    if ((rc = check_arrays({{"norm", norm, 4, false}, {"workspace", workspace, 8, false}}))) return rc;
    int total = 0;
    for (const ClipTable &t : tables) total += clip_groups(t);
    if (workspace_bytes < ((size_t)total + 1) * sizeof(double)) return bad_workspace(((size_t)total + 1) * sizeof(double), workspace_bytes);
    if (tables.empty()) tables.push_back(ClipTable{});
    const hipStream_t st = static_cast<hipStream_t>(stream);
    double *const partials = static_cast<double *>(workspace);
    int at = 0;
    for (const ClipTable &t : tables) {
        if (t.count == 0) continue;
        if ((rc = clip_squares(t, clip_groups(t), partials + at, st))) return rc;
        at += clip_groups(t);
    }
    for (const ClipTable &t : tables)
        if ((rc = clip_scale(t, t.count == 0 ? 1 : clip_groups(t), partials, total, max_norm, norm, st))) return rc;
    return T2FW_OK;
} catch (const std::exception &e) {
    return fail(T2FW_ERR_UNSUPPORTED, "clipping: %s", e.what());
}

}  // extern "C"
