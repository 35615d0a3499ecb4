// Argument block and host entry points of the selective state space scan (select_fwd.hip, select_bwd.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

constexpr int SELECT_STATES = 64;       // states of a channel, at most
constexpr int SELECT_TILE = 16;         // steps from checkpoint to checkpoint

struct SelectArgs {
    const void *x, *dt, *b, *c, *gate;  // [B, T, D], [B, T, N] for b and c; the last axis dense; gate may be null
    const void *g_y;                    // [B, T, D]
    const float *a, *skip, *dt_bias;    // [D, N], [D] or null
    const float *s0, *g_state;          // [B, D, N] or null
    const void *lengths;                // [B] int32 / int64, or null: every row has T steps
    void *y;                            // [B, T, D] dense
    float *last;                        // [B, D, N]
    float *ckpt;                        // state before every tile [B, tiles, D, padded N], or null
    float *maps;                        // scratch: the chunks' maps [chunks, B, D, padded N], and the sums of their steps' lengths [chunks, B, D]
    void *d_x, *d_dt, *d_b, *d_c, *d_gate;
    float *d_a, *d_skip, *d_bias, *d_s0;     // d_skip, d_bias, d_s0 may be null
    float *bc, *sums;                   // scratch: gradients of b and c by blocks of channels (G^2 / 8 bytes a channel and step, of G lanes a channel: 2 for 16
                                        // states, 32 for 64); of a, skip and dt_bias by rows and chunks
    int64_t B, T, D, N;
    // strides of rows and steps, in elements
    int64_t x_b, x_t, dt_b, dt_t, b_b, b_t, c_b, c_t, z_b, z_t, g_b, g_t;
    int32_t softplus, wide_lengths;
};

struct SelectPlan {
    size_t checkpoints, forward, backward;       // bytes
};

SelectPlan select_plan(int64_t B, int64_t T, int64_t D, int64_t N);
int select_forward(const SelectArgs &a, int dtype, hipStream_t stream);
int select_backward(const SelectArgs &a, int dtype, hipStream_t stream);
int select_step(const SelectArgs &a, int dtype, hipStream_t stream);

}  // namespace t2fw
