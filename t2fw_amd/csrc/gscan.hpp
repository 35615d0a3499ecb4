// Argument blocks and host entry points of the per-channel recurrence (gscan.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

struct GscanArgs {
    const void *x, *f, *g_out;          // [B, T, D]; strides below, the last axis dense
    const void *s0, *g_state;           // [B, D] in the accumulators' type
    void *out, *final_state;            // forward: h [B, T, D] dense, the last state [B, D]
    void *d_x, *d_f, *d_s0;             // backward: dense
    void *ckpt;                         // state before every chunk (gscan.hip), or null
    void *words;                        // scratch: the chunks' maps
    const void *lengths;                // [B] int32 / int64, or null: every row has T steps
    int64_t B, T, D;
    int64_t x_b, x_t, f_b, f_t, g_b, g_t;    // strides of batch rows and steps, in elements
    int32_t wide_lengths, logits;       // lengths are int64; f holds gate logits
    int32_t looks;                      // of a chunk at what another hands on, before it does without
};

struct GscanPlan {
    size_t checkpoints, workspace;      // bytes
};

GscanPlan gscan_plan(int64_t B, int64_t T, int64_t D, int dtype);
int gscan_forward(const GscanArgs &a, int dtype, hipStream_t stream);
int gscan_backward(const GscanArgs &a, int dtype, hipStream_t stream);
int gscan_step(const GscanArgs &a, int dtype, hipStream_t stream);

}  // namespace t2fw
