// Argument block and host entry points of the short causal convolution (short_conv.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

constexpr int CONV_TAPS = 8;            // at most; at least 2

struct ConvArgs {
    const void *x, *g_y;                // [B, T, D]; strides below, the last axis dense
    const void *w, *bias;               // [D, taps], [D] or null
    const void *state, *g_last;         // [B, taps - 1, D], or null
    const void *lengths;                // [B] int32 / int64, or null: every row has T steps
    void *y, *last;                     // forward: [B, T, D] dense, [B, taps - 1, D]
    void *d_x, *d_w, *d_bias, *d_state; // backward: dense; d_bias and d_state may be null
    float *partials;                    // backward: conv_partials() rows of D (taps + 1) sums
    int64_t B, T, D;
    int64_t x_b, x_t, g_b, g_t;         // strides of batch rows and steps, in elements
    int32_t taps, silu, wide_lengths, wide_w;
};

int64_t conv_partials(int64_t B, int64_t T, int64_t D, int taps, int dtype);
int conv_forward(const ConvArgs &a, int dtype, hipStream_t stream);
int conv_backward(const ConvArgs &a, int dtype, hipStream_t stream);
int conv_step(const ConvArgs &a, int dtype, hipStream_t stream);

}  // namespace t2fw
