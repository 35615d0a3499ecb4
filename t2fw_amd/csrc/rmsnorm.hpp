// Argument blocks and host entry points of the residual's addition and root-mean-square norm (rmsnorm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

struct NormArgs {
    const void *x, *res, *w;            // [N, D] of the tensors' type, [N, D] of the stream's (or null), [D]
    const void *g_y, *g_res;            // gradients of y and of the stream (either or null)
    void *y, *stored;                   // forward results; `stored` is x + res in the stream's type
    void *q;                            // instead of y: float8 e4m3
    float *scales;                      // [N, groups]
    void *d_x, *d_res;                  // backward results; d_res is null where it is d_x
    void *d_w;                          // [D] of w's type
    void *partials;                     // [norm_partials(N, D), D], the workgroups' shares of d_w, in the accumulators' type
    int64_t N, D, group, groups;        // group: columns of one scale
    double eps;
    int32_t wide_stream, wide_w;        // the stream / the weights are float32 next to 16-bit tensors
};

int64_t norm_partials(int64_t N, int64_t D);
int norm_forward(const NormArgs &a, int dtype, hipStream_t stream);
int norm_backward(const NormArgs &a, int dtype, hipStream_t stream);

}  // namespace t2fw
