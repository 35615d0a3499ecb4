// Argument blocks and host entry points of the clipped policy loss (policy_loss.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

constexpr int POLICY_SUMS = 8192;               // workgroups of a launch, at most

struct PolicyLossArgs {
    const void *logits;                          // [N, V]
    const int64_t *targets;                      // [N]
    const float *old_logp, *ref_logp, *adv;      // [N]
    const uint8_t *mask;                         // [N], or null: every token counts
    float *loss, *logp, *tops, *coef;            // [1], [N], [N, 2], [N]: what the backward needs are the last two
    int64_t *tokens;                             // [1] scratch: the tokens that count
    double *sums;                                // [POLICY_SUMS] scratch: the workgroups' shares of the loss
    void *d_logits;                              // [N, V], or null: no gradient now
    const float *g_loss;                         // backward: the gradient of the loss, one value on the device
    int64_t N, V;
    float low, high, kl, scale;                  // ratios are held in [low, high]; factor of the loss
    int32_t unless_one;                          // backward: d_logits holds the gradient for g_loss = 1 already
};

int policy_loss_forward(const PolicyLossArgs &a, int dtype, hipStream_t stream);
int policy_loss_backward(const PolicyLossArgs &a, int dtype, hipStream_t stream);

}  // namespace t2fw
