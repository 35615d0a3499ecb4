// C ABI of the selective state space layer and of beam search (include/t2fw_hip.h): argument validation, and what a call needs laid out.
#include "checks.hpp"
#include "beam.hpp"
#include "select.hpp"
#include "short_conv.hpp"

#include <exception>
#include <vector>

namespace t2fw {
namespace {

int check_lowp(int32_t dtype, const char *what) {
    if (dtype != T2FW_F32 && dtype != T2FW_F16 && dtype != T2FW_BF16)
        return fail(T2FW_ERR_BAD_DTYPE, "%s: fp32, fp16 or bf16 (dtype code %d)", what, dtype);
    return T2FW_OK;
}

int check_conv(int64_t B, int64_t T, int64_t D, int64_t taps, int32_t dtype, int32_t flags) {
    int rc = check_lowp(dtype, "short convolution");
    if (rc || (rc = check_sizes({B, T, D, CONV_TAPS + 1}, "short convolution"))) return rc;
    if (D < 1) return fail(T2FW_ERR_BAD_SHAPE, "short convolution: at least one channel");
    if (taps < 2 || taps > CONV_TAPS) return fail(T2FW_ERR_BAD_SHAPE, "short convolution: 2 to %d taps, not %lld", CONV_TAPS, (long long)taps);
    if (flags & ~(T2FW_CONV_SILU | T2FW_CONV_LENGTHS64 | T2FW_CONV_WEIGHT_F32)) return fail(T2FW_ERR_UNSUPPORTED, "short convolution: unknown flags %d", flags);
    return T2FW_OK;
}
// strides in elements: of rows and steps, or null for dense arrays
int conv_args(ConvArgs &a, int64_t B, int64_t T, int64_t D, int64_t taps, const int64_t *strides, bool backward, int32_t dtype, int32_t flags) {
    a.B = B; a.T = T; a.D = D;
    a.taps = (int32_t)taps;
    a.silu = (flags & T2FW_CONV_SILU) != 0;
    a.wide_lengths = (flags & T2FW_CONV_LENGTHS64) != 0;
    a.wide_w = dtype == T2FW_F32 || (flags & T2FW_CONV_WEIGHT_F32) != 0;
    a.x_b = a.g_b = T * D;
    a.x_t = a.g_t = D;
    if (strides == nullptr) return T2FW_OK;
    for (int i = 0; i < (backward ? 4 : 2); ++i)
        if (strides[i] < 0) return fail(T2FW_ERR_BAD_SHAPE, "short convolution: strides must be non-negative");
    a.x_b = strides[0]; a.x_t = strides[1];
    if (backward) {
        a.g_b = strides[2]; a.g_t = strides[3];
    }
    return T2FW_OK;
}
size_t conv_weight_size(int32_t dtype, int32_t flags) { return flags & T2FW_CONV_WEIGHT_F32 ? 4 : size_of(dtype); }
size_t lengths_size(bool wide) { return wide ? 8 : 4; }

int check_select(int64_t B, int64_t T, int64_t D, int64_t N, int32_t dtype, int32_t flags) {
    int rc = check_lowp(dtype, "selective scan");
    if (rc || (rc = check_sizes({B, T, D, 2 * SELECT_STATES}, "selective scan"))) return rc;
    if (D < 1) return fail(T2FW_ERR_BAD_SHAPE, "selective scan: at least one channel");
    if (N < 1 || N > SELECT_STATES) return fail(T2FW_ERR_BAD_SHAPE, "selective scan: 1 to %d states of a channel, not %lld", SELECT_STATES, (long long)N);
    if (flags & ~(T2FW_SELECT_SOFTPLUS | T2FW_SELECT_LENGTHS64)) return fail(T2FW_ERR_UNSUPPORTED, "selective scan: unknown flags %d", flags);
    return T2FW_OK;
}
// rows and steps of x, dt, b, c, gate and, backward, g_y
int select_args(SelectArgs &s, int64_t B, int64_t T, int64_t D, int64_t N, const int64_t *strides, bool backward, size_t es, int32_t flags) {
    s.B = B; s.T = T; s.D = D; s.N = N;
    s.softplus = (flags & T2FW_SELECT_SOFTPLUS) != 0;
    s.wide_lengths = (flags & T2FW_SELECT_LENGTHS64) != 0;
    int64_t *const to[12] = {&s.x_b, &s.x_t, &s.dt_b, &s.dt_t, &s.b_b, &s.b_t, &s.c_b, &s.c_t, &s.z_b, &s.z_t, &s.g_b, &s.g_t};
    for (int i = 0; i < 12; ++i) {
        const int64_t width = i >= 4 && i < 8 ? N : D;
        *to[i] = i % 2 == 0 ? T * width : width;
        if (strides == nullptr || (i >= 10 && !backward) || (i / 2 == 4 && s.gate == nullptr)) continue;
        if (strides[i] < 0) return fail(T2FW_ERR_BAD_SHAPE, "selective scan: strides must be non-negative");
        // (a tile of 16 steps is addressed by 32 bits)
        if (i % 2 == 1 && T > 1 && strides[i] > (int64_t)(0xffffffffu / (SELECT_TILE * es)))
            return fail(T2FW_ERR_UNSUPPORTED, "selective scan: steps are %lld elements apart, 16 of them have to be within 4 GB", (long long)strides[i]);
        *to[i] = strides[i];
    }
    return T2FW_OK;
}

struct BeamLayout {
    BeamPieces cut;
    int64_t shares;                          // bytes of the first array of the scratch
    size_t bytes;
};
BeamLayout beam_layout(int64_t B, int64_t K, int64_t V, int64_t n) {
    BeamLayout l;
    l.cut = beam_pieces(B, K, V, n);
    l.shares = B * K * l.cut.pieces * 16;
    l.bytes = (size_t)(l.shares + B * K * l.cut.pieces * n * 8);
    return l;
}
int check_beams(int64_t B, int64_t K, int64_t V, int64_t n, int32_t dtype) {
    int rc = check_lowp(dtype, "beam selection");
    if (rc || (rc = check_sizes({B, K, V, BEAM_COUNT}, "beam selection"))) return rc;
    if (K < 1 || K > BEAM_ROWS) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: 1 to %d beams, not %lld", BEAM_ROWS, (long long)K);
    if (V < 1 || K * V > 0x7fffffff) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: %lld x %lld candidates", (long long)K, (long long)V);
    if (n < 1 || n > BEAM_COUNT) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: 1 to %d candidates, not %lld", BEAM_COUNT, (long long)n);
    if (n > K * V) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: %lld of %lld candidates", (long long)n, (long long)(K * V));
    return T2FW_OK;
}

}  // namespace
}  // namespace t2fw

using namespace t2fw;

extern "C" {

int t2fw_short_conv_forward(const void *x, const void *w, const void *bias, const void *s0, const void *lengths, void *y, void *last,
                            int64_t B, int64_t T, int64_t D, int64_t taps, const int64_t *strides, int32_t dtype, int32_t flags, void *stream) {
    int rc = check_conv(B, T, D, taps, dtype, flags);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    const size_t es = size_of(dtype), ws = conv_weight_size(dtype, flags);
    if ((rc = check_arrays({{"x", x, es, T == 0}, {"w", w, ws, false}, {"bias", bias, ws, true}, {"s0", s0, es, true},
                            {"lengths", lengths, lengths_size(flags & T2FW_CONV_LENGTHS64), true}, {"y", y, es, T == 0}, {"last", last, es, false}})))
        return rc;
    ConvArgs a{};
    if ((rc = conv_args(a, B, T, D, taps, strides, false, dtype, flags))) return rc;
    a.x = x; a.w = w; a.bias = bias; a.state = s0; a.lengths = lengths; a.y = y; a.last = last;
    return conv_forward(a, dtype, static_cast<hipStream_t>(stream));
}

size_t t2fw_short_conv_backward_workspace_bytes(int64_t B, int64_t T, int64_t D, int64_t taps, int32_t dtype) {
    if (check_conv(B, T, D, taps, dtype, 0)) return 0;
    return (size_t)(conv_partials(B, T, D, (int)taps, dtype) * D * (taps + 1)) * sizeof(float);
}

int t2fw_short_conv_backward(const void *g_y, const void *g_last, const void *x, const void *w, const void *bias, const void *s0, const void *lengths,
                             void *d_x, void *d_w, void *d_bias, void *d_s0, int64_t B, int64_t T, int64_t D, int64_t taps, const int64_t *strides,
                             int32_t dtype, int32_t flags, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_conv(B, T, D, taps, dtype, flags);
    if (rc) return rc;
    const bool none = B == 0 || T == 0;
    const size_t es = size_of(dtype), ws = conv_weight_size(dtype, flags), need = t2fw_short_conv_backward_workspace_bytes(B, T, D, taps, dtype);
    if ((rc = check_arrays({{"g_y", g_y, es, none}, {"g_last", g_last, es, true}, {"x", x, es, none}, {"w", w, ws, false}, {"bias", bias, ws, true},
                            {"s0", s0, es, true}, {"lengths", lengths, lengths_size(flags & T2FW_CONV_LENGTHS64), true}, {"d_x", d_x, es, none},
                            {"d_w", d_w, ws, false}, {"d_bias", d_bias, ws, true}, {"d_s0", d_s0, es, true}, {"workspace", workspace, 16, need == 0}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    ConvArgs a{};
    if ((rc = conv_args(a, B, T, D, taps, strides, true, dtype, flags))) return rc;
    a.g_y = g_y; a.g_last = g_last; a.x = x; a.w = w; a.bias = bias; a.state = s0; a.lengths = lengths;
    a.d_x = d_x; a.d_w = d_w; a.d_bias = d_bias; a.d_state = d_s0;
    a.partials = static_cast<float *>(workspace);
    return conv_backward(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_short_conv_step(const void *x, const void *w, const void *bias, const void *s0, void *y, void *next_state, int64_t B, int64_t D, int64_t taps,
                         int64_t x_stride, int32_t dtype, int32_t flags, void *stream) {
    int rc = check_conv(B, 1, D, taps, dtype, flags & ~T2FW_CONV_LENGTHS64);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    if (x_stride < 0) return fail(T2FW_ERR_BAD_SHAPE, "short convolution: strides must be non-negative");
    const size_t es = size_of(dtype), ws = conv_weight_size(dtype, flags);
    if ((rc = check_arrays({{"x", x, es, false}, {"w", w, ws, false}, {"bias", bias, ws, true}, {"s0", s0, es, false}, {"y", y, es, false},
                            {"next_state", next_state, es, false}})))
        return rc;
    ConvArgs a{};
    if ((rc = conv_args(a, B, 1, D, taps, nullptr, false, dtype, flags))) return rc;
    a.x = x; a.w = w; a.bias = bias; a.state = s0; a.y = y; a.last = next_state;
    a.x_b = x_stride;
    return conv_step(a, dtype, static_cast<hipStream_t>(stream));
}

size_t t2fw_selective_scan_checkpoint_bytes(int64_t B, int64_t T, int64_t D, int64_t N) {
    return check_select(B, T, D, N, T2FW_F32, 0) ? 0 : select_plan(B, T, D, N).checkpoints;
}
size_t t2fw_selective_scan_workspace_bytes(int64_t B, int64_t T, int64_t D, int64_t N) {
    return check_select(B, T, D, N, T2FW_F32, 0) ? 0 : select_plan(B, T, D, N).forward;
}
size_t t2fw_selective_scan_backward_workspace_bytes(int64_t B, int64_t T, int64_t D, int64_t N) {
    return check_select(B, T, D, N, T2FW_F32, 0) ? 0 : select_plan(B, T, D, N).backward;
}

int t2fw_selective_scan_forward(const void *x, const void *dt, const float *a, const void *b, const void *c, const float *skip, const void *gate,
                                const float *dt_bias, const float *s0, const void *lengths, void *y, float *last, void *ckpt, int64_t B, int64_t T,
                                int64_t D, int64_t N, const int64_t *strides, int32_t dtype, int32_t flags, void *workspace, size_t workspace_bytes,
                                void *stream) {
    int rc = check_select(B, T, D, N, dtype, flags);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    const size_t es = size_of(dtype), need = t2fw_selective_scan_workspace_bytes(B, T, D, N);
    const bool none = T == 0;
    if ((rc = check_arrays({{"x", x, es, none}, {"dt", dt, es, none}, {"a", a, 4, false}, {"b", b, es, none}, {"c", c, es, none}, {"skip", skip, 4, true},
                            {"gate", gate, es, true}, {"dt_bias", dt_bias, 4, true}, {"s0", s0, 4, true},
                            {"lengths", lengths, lengths_size(flags & T2FW_SELECT_LENGTHS64), true}, {"y", y, es, none}, {"last", last, 4, false},
                            {"ckpt", ckpt, 16, true}, {"workspace", workspace, 16, need == 0}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    SelectArgs s{};
    s.x = x; s.dt = dt; s.a = a; s.b = b; s.c = c; s.skip = skip; s.gate = gate; s.dt_bias = dt_bias; s.s0 = s0; s.lengths = lengths;
    s.y = y; s.last = last; s.ckpt = static_cast<float *>(ckpt); s.maps = static_cast<float *>(workspace);
    if ((rc = select_args(s, B, T, D, N, strides, false, es, flags))) return rc;
    return select_forward(s, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_selective_scan_backward(const void *g_y, const float *g_last, const void *x, const void *dt, const float *a, const void *b, const void *c,
                                 const float *skip, const void *gate, const float *dt_bias, const void *lengths, const void *ckpt, void *d_x, void *d_dt,
                                 float *d_a, void *d_b, void *d_c, float *d_skip, void *d_gate, float *d_bias, float *d_s0, int64_t B, int64_t T,
                                 int64_t D, int64_t N, const int64_t *strides, int32_t dtype, int32_t flags, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    int rc = check_select(B, T, D, N, dtype, flags);
    if (rc) return rc;
    const size_t es = size_of(dtype), need = t2fw_selective_scan_backward_workspace_bytes(B, T, D, N);
    const bool none = B == 0 || T == 0;
    if ((rc = check_arrays({{"g_y", g_y, es, none}, {"g_last", g_last, 4, true}, {"x", x, es, none}, {"dt", dt, es, none}, {"a", a, 4, false},
                            {"b", b, es, none}, {"c", c, es, none}, {"skip", skip, 4, true}, {"gate", gate, es, true}, {"dt_bias", dt_bias, 4, true},
                            {"lengths", lengths, lengths_size(flags & T2FW_SELECT_LENGTHS64), true}, {"ckpt", ckpt, 16, none}, {"d_x", d_x, es, none},
                            {"d_dt", d_dt, es, none}, {"d_a", d_a, 4, false}, {"d_b", d_b, es, none}, {"d_c", d_c, es, none}, {"d_skip", d_skip, 4, true},
                            {"d_gate", d_gate, es, gate == nullptr || none}, {"d_bias", d_bias, 4, true}, {"d_s0", d_s0, 4, true},
                            {"workspace", workspace, 16, need == 0}})))
        return rc;
    if (workspace_bytes < need) return bad_workspace(need, workspace_bytes);
    SelectArgs s{};
    s.g_y = g_y; s.g_state = g_last; s.x = x; s.dt = dt; s.a = a; s.b = b; s.c = c; s.skip = skip; s.gate = gate; s.dt_bias = dt_bias; s.lengths = lengths;
    s.ckpt = static_cast<float *>(const_cast<void *>(ckpt)); s.maps = static_cast<float *>(workspace);
    s.d_x = d_x; s.d_dt = d_dt; s.d_a = d_a; s.d_b = d_b; s.d_c = d_c; s.d_skip = d_skip; s.d_gate = d_gate; s.d_bias = d_bias; s.d_s0 = d_s0;
    if ((rc = select_args(s, B, T, D, N, strides, true, es, flags))) return rc;
    return select_backward(s, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_selective_scan_step(const void *x, const void *dt, const float *a, const void *b, const void *c, const float *skip, const void *gate,
                             const float *dt_bias, const float *s0, void *y, float *next_state, int64_t B, int64_t D, int64_t N, const int64_t *strides,
                             int32_t dtype, int32_t flags, void *stream) {
    int rc = check_select(B, 1, D, N, dtype, flags & ~T2FW_SELECT_LENGTHS64);
    if (rc) return rc;
    if (B == 0) return T2FW_OK;
    const size_t es = size_of(dtype);
    if ((rc = check_arrays({{"x", x, es, false}, {"dt", dt, es, false}, {"a", a, 4, false}, {"b", b, es, false}, {"c", c, es, false},
                            {"skip", skip, 4, true}, {"gate", gate, es, true}, {"dt_bias", dt_bias, 4, true}, {"s0", s0, 4, false}, {"y", y, es, false},
                            {"next_state", next_state, 4, false}})))
        return rc;
    SelectArgs s{};
    s.x = x; s.dt = dt; s.a = a; s.b = b; s.c = c; s.skip = skip; s.gate = gate; s.dt_bias = dt_bias; s.s0 = s0; s.y = y; s.last = next_state;
    int64_t both[10];
    for (int i = 0; strides != nullptr && i < 10; ++i) both[i] = strides[i / 2];         // (there is one step)
    if ((rc = select_args(s, B, 1, D, N, strides == nullptr ? nullptr : both, false, es, flags))) return rc;
    return select_step(s, dtype, static_cast<hipStream_t>(stream));
}

size_t t2fw_beam_select_workspace_bytes(int64_t B, int64_t K, int64_t V, int64_t n, int32_t dtype) {
    if (check_beams(B, K, V, n, dtype)) return 0;
    return beam_layout(B, K, V, n).bytes;
}

int t2fw_beam_select(const void *logits, const float *scores, const void *finished, float *out_scores, int64_t *out_beams, int64_t *out_tokens,
                     int64_t B, int64_t K, int64_t V, int64_t n, int64_t pad, int32_t dtype, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_beams(B, K, V, n, dtype);
    if (rc) return rc;
    if (finished != nullptr && (pad < 0 || pad >= V)) return fail(T2FW_ERR_BAD_SHAPE, "beam selection: the token of ended beams is %lld of %lld", (long long)pad, (long long)V);
    if (B == 0) return T2FW_OK;
    const BeamLayout l = beam_layout(B, K, V, n);
    if ((rc = check_arrays({{"logits", logits, size_of(dtype), false}, {"scores", scores, 4, false}, {"finished", finished, 1, true},
                            {"out_scores", out_scores, 4, false}, {"out_beams", out_beams, 8, false}, {"out_tokens", out_tokens, 8, false},
                            {"workspace", workspace, 16, false}})))
        return rc;
    if (workspace_bytes < l.bytes) return bad_workspace(l.bytes, workspace_bytes);
    BeamArgs a{};
    a.logits = logits; a.scores = scores; a.finished = static_cast<const uint8_t *>(finished);
    a.out_scores = out_scores; a.out_beams = out_beams; a.out_tokens = out_tokens;
    a.partial = workspace;
    a.lists = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + l.shares);
    a.B = B; a.K = K; a.V = V; a.n = (int32_t)n; a.pieces = l.cut.pieces; a.piece = l.cut.piece; a.pad = (int32_t)pad;
    return beam_select(a, dtype, static_cast<hipStream_t>(stream));
}

int t2fw_beam_reorder(const t2fw_reorder_desc *arrays, int64_t count, const int64_t *beams, int64_t B, int64_t K, void *stream) try {
    int rc = check_sizes({B, K}, "reordering");
    if (rc) return rc;
    if (K < 1 || K > REORDER_BEAMS) return fail(T2FW_ERR_BAD_SHAPE, "reordering: 1 to %d beams, not %lld", REORDER_BEAMS, (long long)K);
    if (count < 0 || count > 0x7fffffff) return fail(T2FW_ERR_BAD_SHAPE, "reordering: %lld arrays", (long long)count);
    if (count > 0 && arrays == nullptr) return fail(T2FW_ERR_NULL_POINTER, "null array list");
    if (B == 0 || count == 0) return T2FW_OK;
    if ((rc = check_arrays({{"beams", beams, 8, false}}))) return rc;
    constexpr int64_t MOST = (1ll << 32) / 256 - 1;                  // workgroups of a launch
    const int64_t piece = reorder_piece(K);
    std::vector<ReorderTable> tables;
    for (int64_t i = 0; i < count; ++i) {
        const t2fw_reorder_desc &d = arrays[i];
        if ((rc = check_sizes({B, K, d.row_bytes}, "reordering"))) return rc;
        if (d.row_bytes == 0) continue;
        if ((rc = check_arrays({{"src", d.src, 1, false}, {"dst", d.dst, 1, false}}))) return rc;
        const int64_t per = (d.row_bytes + piece - 1) / piece;
        if (per > MOST || B > MOST / per) return fail(T2FW_ERR_BAD_SHAPE, "reordering: too many workgroups for one launch");
        if (tables.empty() || tables.back().count == REORDER_TABLE || tables.back().pieces + per * B > MOST) tables.push_back(ReorderTable{});
        ReorderTable &t = tables.back();
        t.src[t.count] = static_cast<const char *>(d.src);
        t.dst[t.count] = static_cast<char *>(d.dst);
        t.row[t.count] = d.row_bytes;
        t.first[t.count] = t.pieces;
        t.pieces += (uint32_t)(per * B);
        ++t.count;
    }
    for (const ReorderTable &t : tables)
        if ((rc = beam_reorder(t, beams, B, K, static_cast<hipStream_t>(stream)))) return rc;
    return T2FW_OK;
} catch (const std::exception &e) {
    return fail(T2FW_ERR_UNSUPPORTED, "reordering: %s", e.what());
}

}  // extern "C"
